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
// token at a time, a lane's 16 latent values are two 16-byte loads, a 128-dim
// block is eight lanes (three shuffles for its maximum) and lane i turns pair i,
// whose turn fraction it keeps.
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

__device__ __forceinline__ uint32_t pack_e4m3(float2 a, float2 b) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, __NV_E4M3) |
         ((uint32_t)__nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, __NV_E4M3) << 16);
}

__device__ __forceinline__ unsigned long long pack_f32x2(float a, float b) {
  unsigned long long v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}

// Minus the quotients of a word's two BF16 values by the scale; n is minus its reciprocal.
__device__ __forceinline__ float2 quotient2(uint32_t w, unsigned long long scale, unsigned long long n) {
  const unsigned long long x = pack_f32x2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  unsigned long long y, r;
  float2 z;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(x), "l"(n));
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(y), "l"(scale), "l"(x));
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y) : "l"(r), "l"(n), "l"(y));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(z.x), "=f"(z.y) : "l"(y));
  return z;
}

// One token's row as a lane holds it.
struct Row {
  uint4 v0, v1;          // 16 latent values
  __nv_bfloat16 r0, r1;  // a pair of rope values
  int32_t pos;
};

// kWide: kv rows start on 16-byte boundaries.
template <bool kWide>
__device__ __forceinline__ void load_row(const AppendParams& p, uint32_t t, int lane, int e0, int e1, Row& r) {
  const uint32_t b = p.queries != 0 ? t / (uint32_t)p.queries : 0, s = t - b * (uint32_t)p.queries;
  const __nv_bfloat16* const kr = p.k_rope + b * p.krs[0] + s * p.krs[1];
  load16<kWide>(p.kv + b * p.kvs[0] + s * p.kvs[1] + lane * 16, r.v0, r.v1);
  r.r0 = kr[e0];
  r.r1 = kr[e1];
  r.pos = p.positions != nullptr ? __ldg(p.positions + t) : 0;
}

template <bool kFp8>
__device__ __forceinline__ void write_row(const AppendParams& p, long long slot, int lane, int e0, int e1,
                                          unsigned long long fraction, Row& r) {
  if (p.inv_freq != nullptr) {
    float c, sn;
    rotary_cos_sin(r.pos, fraction, p.factor, 1.f, &c, &sn);
    const float2 turned = rotate_pair(__bfloat162float(r.r0), __bfloat162float(r.r1), c, sn);
    r.r0 = __float2bfloat16_rn(turned.x);
    r.r1 = __float2bfloat16_rn(turned.y);
  }
  __nv_bfloat16* rope;
  if (kFp8) {
    uint8_t* const row = p.cache + slot * kApRowBytes;
    const uint32_t w[8] = {r.v0.x, r.v0.y, r.v0.z, r.v0.w, r.v1.x, r.v1.y, r.v1.z, r.v1.w};
    // |bits| order as the magnitudes do, a NaN above every number
    uint32_t both = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) both = __vmaxu2(both, w[k] & 0x7fff7fffu);
    uint32_t top = max(both & 0xffffu, both >> 16);
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
    const float amax = __uint_as_float(top << 16);
    float scale;
    // kv / scale, correctly rounded: with the correctly rounded reciprocal one
    // Newton step on the quotient's exact remainder gives it (Markstein, 1990)
    // while nothing leaves the normal range; 16 divisions would cost a lane
    // more than all the rest. Two values go through an instruction, negated:
    // so an exact quotient's zero remainder leaves a zero its sign.
    uint32_t q[4];
    if (top < 0x7f80u && amax >= 0x1p-60f && amax <= 0x1p60f) {  // every value finite
      constexpr float kInv = 1.f / 448.f;
      scale = __fmul_rn(amax, kInv);
      scale = __fmaf_rn(__fmaf_rn(scale, -448.f, amax), kInv, scale);
      const float inv = __frcp_rn(scale);
      const unsigned long long s2 = pack_f32x2(scale, scale), n2 = pack_f32x2(-inv, -inv);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        q[k] = pack_e4m3(quotient2(w[2 * k], s2, n2), quotient2(w[2 * k + 1], s2, n2)) ^ 0x80808080u;
      }
    } else {
      scale = amax > 0.f ? __fdiv_rn(amax, 448.f) : 1.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float x[4] = {__fdiv_rn(__uint_as_float(w[2 * k] << 16), scale),
                            __fdiv_rn(__uint_as_float(w[2 * k] & 0xffff0000u), scale),
                            __fdiv_rn(__uint_as_float(w[2 * k + 1] << 16), scale),
                            __fdiv_rn(__uint_as_float(w[2 * k + 1] & 0xffff0000u), scale)};
        q[k] = pack_e4m3(make_float2(x[0], x[1]), make_float2(x[2], x[3]));
      }
    }
    reinterpret_cast<uint4*>(row)[lane] = make_uint4(q[0], q[1], q[2], q[3]);
    if ((lane & 7) == 0) reinterpret_cast<float*>(row + kDimLatent)[lane >> 3] = scale;
    rope = reinterpret_cast<__nv_bfloat16*>(row + kDimLatent + 16);
  } else {
    uint4* const dst = reinterpret_cast<uint4*>(p.kv_cache + slot * kDimLatent) + 2 * lane;
    dst[0] = r.v0;
    dst[1] = r.v1;
    rope = p.rope_cache + slot * kDimRope;
  }
  if (e1 == e0 + 1) {
    __nv_bfloat162 pair;
    pair.x = r.r0;
    pair.y = r.r1;
    *reinterpret_cast<__nv_bfloat162*>(rope + e0) = pair;
  } else {
    rope[e0] = r.r0;
    rope[e1] = r.r1;
  }
}

// A warp walks over tokens, the next token's slot under way. Measured with FP8
// rows: 151552 tokens 47.4 us (5.8 TB/s, near the copy rate), 32768 tokens
// 12.3, 65536 of which half are padding 14.9 (warps meet unequal numbers of
// those). Six blocks an SM, all of them resident, hide the loads; eight took
// 50.3, 12.9 and 14.8, and two rounds of eight 15.3 for the last. Keeping the
// next token's row in registers too (five blocks) was slower.
constexpr int kApBlocks = 6;

template <bool kFp8, bool kWide>
__global__ void __launch_bounds__(kApThreads, kApBlocks) append_kernel(const AppendParams p) {
  const int lane = threadIdx.x & 31;
  const uint32_t stride = gridDim.x * (kApThreads / 32);
  const uint32_t tokens = (uint32_t)p.tokens;  // < 2^31
  const int e0 = p.half ? lane : 2 * lane, e1 = p.half ? lane + 32 : 2 * lane + 1;
  const unsigned long long fraction = p.inv_freq != nullptr ? turn_fraction(__ldg(p.inv_freq + lane)) : 0;
  uint32_t t = blockIdx.x * (kApThreads / 32) + (threadIdx.x >> 5);
  int32_t next = t < tokens ? __ldg(p.slots + t) : -1;
  for (; t < tokens; t += stride) {
    const int32_t slot = next;
    next = t + stride < tokens ? __ldg(p.slots + t + stride) : -1;
    if (slot < 0 || slot >= p.rows) continue;
    Row row;
    load_row<kWide>(p, t, lane, e0, e1, row);
    write_row<kFp8>(p, slot, lane, e0, e1, fraction, row);
  }
}

}  // namespace

cudaError_t launch_append_kv(const AppendParams& p, cudaStream_t stream) {
  long long blocks = (p.tokens + kApThreads / 32 - 1) / (kApThreads / 32);
  if (blocks > 148 * kApBlocks) blocks = 148 * kApBlocks;
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
