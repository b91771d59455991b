// Cache append: the new tokens' latent rows and (turned) rope rows into the
// cache rows that their slots name.
//   BF16 cache: kv_cache[slot] = kv, rope_cache[slot] = R(position) k_rope
//   FP8 cache:  the 656-byte row of fp8.cu, scale k = max |kv| over latent
//               dims [128k, 128k + 128) / 448 (1 for an all-zero block),
//               values e4m3(kv / scale) with both quotients rounded to FP32,
//               the same bits as quantize_kv_fp8 on the host.
// A slot outside [0, rows) writes nothing (padding). Slots of one call are
// distinct (a page plan's are).
//
// Bound: HBM, 1152 bytes read and 1152 (656) written per token; one warp per
// token, a lane's 16 latent values are two 16-byte loads, a 128-dim block is
// eight lanes (three shuffles for its maximum) and lane i turns pair i.
#include <cuda_fp8.h>

#include "serving.cuh"

namespace dsa {
namespace {

constexpr int kApRowBytes = 656;
constexpr int kApThreads = 256;

template <bool kWide>
__device__ __forceinline__ void load16(const __nv_bfloat16* src, uint4& a, uint4& b) {
  if (kWide) {
    a = __ldg(reinterpret_cast<const uint4*>(src));
    b = __ldg(reinterpret_cast<const uint4*>(src) + 1);
  } else {
    const unsigned short* s = reinterpret_cast<const unsigned short*>(src);
    uint32_t r[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) r[k] = (uint32_t)s[2 * k] | ((uint32_t)s[2 * k + 1] << 16);
    a = make_uint4(r[0], r[1], r[2], r[3]);
    b = make_uint4(r[4], r[5], r[6], r[7]);
  }
}

// kWide: kv rows start on 16-byte boundaries.
template <bool kFp8, bool kWide>
__global__ void __launch_bounds__(kApThreads) append_kernel(const AppendParams p) {
  const int lane = threadIdx.x & 31;
  const long long stride = (long long)gridDim.x * (kApThreads / 32);
  // this lane's pair of rope dims and its frequency
  const int e0 = p.half ? lane : 2 * lane, e1 = p.half ? lane + 32 : 2 * lane + 1;
  const double freq = p.inv_freq != nullptr ? __ldg(p.inv_freq + lane) : 0.0;
  for (long long t = (long long)blockIdx.x * (kApThreads / 32) + (threadIdx.x >> 5); t < p.tokens; t += stride) {
    const long long slot = __ldg(p.slots + t);
    if (slot < 0 || slot >= p.rows) continue;
    const int b = (int)(t / p.queries), s = (int)(t - (long long)b * p.queries);
    const __nv_bfloat16* const kv = p.kv + b * p.kvs[0] + s * p.kvs[1];
    const __nv_bfloat16* const kr = p.k_rope + b * p.krs[0] + s * p.krs[1];
    uint4 v0, v1;
    load16<kWide>(kv + lane * 16, v0, v1);
    __nv_bfloat16 r0 = kr[e0], r1 = kr[e1];
    if (p.inv_freq != nullptr) {
      float c, sn;
      rotary_cos_sin(__ldg(p.positions + t), freq, p.factor, 1.f, &c, &sn);
      const float2 turned = rotate_pair(__bfloat162float(r0), __bfloat162float(r1), c, sn);
      r0 = __float2bfloat16_rn(turned.x);
      r1 = __float2bfloat16_rn(turned.y);
    }
    __nv_bfloat16* rope;
    if (kFp8) {
      uint8_t* const row = p.cache + slot * kApRowBytes;
      const uint32_t w[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
      // |bits| order as the magnitudes do, a NaN above every number
      uint32_t top = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) top = max(top, max(w[k] & 0x7fffu, (w[k] >> 16) & 0x7fffu));
#pragma unroll
      for (int d = 1; d < 8; d <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
      const float amax = __uint_as_float(top << 16);
      const float scale = amax > 0.f ? __fdiv_rn(amax, 448.f) : 1.f;
      uint32_t q[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 lo = make_float2(__fdiv_rn(__uint_as_float(w[2 * k] << 16), scale),
                                      __fdiv_rn(__uint_as_float(w[2 * k] & 0xffff0000u), scale));
        const float2 hi = make_float2(__fdiv_rn(__uint_as_float(w[2 * k + 1] << 16), scale),
                                      __fdiv_rn(__uint_as_float(w[2 * k + 1] & 0xffff0000u), scale));
        q[k] = (uint32_t)__nv_cvt_float2_to_fp8x2(lo, __NV_SATFINITE, __NV_E4M3) |
               ((uint32_t)__nv_cvt_float2_to_fp8x2(hi, __NV_SATFINITE, __NV_E4M3) << 16);
      }
      reinterpret_cast<uint4*>(row)[lane] = make_uint4(q[0], q[1], q[2], q[3]);
      if ((lane & 7) == 0) reinterpret_cast<float*>(row + kDimLatent)[lane >> 3] = scale;
      rope = reinterpret_cast<__nv_bfloat16*>(row + kDimLatent + 16);
    } else {
      uint4* const dst = reinterpret_cast<uint4*>(p.kv_cache + slot * kDimLatent) + 2 * lane;
      dst[0] = v0;
      dst[1] = v1;
      rope = p.rope_cache + slot * kDimRope;
    }
    rope[e0] = r0;
    rope[e1] = r1;
  }
}

}  // namespace

cudaError_t launch_append_kv(const AppendParams& p, cudaStream_t stream) {
  long long blocks = (p.tokens + kApThreads / 32 - 1) / (kApThreads / 32);
  if (blocks > 148 * 8 * 4) blocks = 148 * 8 * 4;
  bool wide = (reinterpret_cast<uintptr_t>(p.kv) & 15u) == 0 && p.kvs[0] % 8 == 0 && p.kvs[1] % 8 == 0;
  const unsigned g = (unsigned)blocks;
  if (p.cache != nullptr) {
    if (wide) append_kernel<true, true><<<g, kApThreads, 0, stream>>>(p);
    else append_kernel<true, false><<<g, kApThreads, 0, stream>>>(p);
  } else {
    if (wide) append_kernel<false, true><<<g, kApThreads, 0, stream>>>(p);
    else append_kernel<false, false><<<g, kApThreads, 0, stream>>>(p);
  }
  return cudaGetLastError();
}

}  // namespace dsa
