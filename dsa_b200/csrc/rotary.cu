// Rotary positions: y = x with `rotary_dim` of its `dim` elements turned by
// the token's position,
//   y_a = f (x_a cos t - x_b sin t),  y_b = f (x_b cos t + x_a sin t),
//   t = position * inv_freq[i],  f = the attention factor,
// over the pairs (a, b) = (2i, 2i + 1) (interleaved) or (i, i + rotary_dim/2)
// (half). The other elements are copied. The gradient of y with respect to x
// is the same map with -t, so the backward pass is this kernel again.
//
// Bound: HBM, 2 * dim elements per head row (16384 tokens x 128 heads x 64 BF16:
// 86 us, 6.2 TB/s). The cosines cost ~30 instructions a pair and depend on the
// token alone: a block computes those of its tokens once into shared memory,
// while its first loads are under way, and a thread walks over heads h,
// h + groups, ... with its pairs' cosines in registers. A unit is two 16-byte
// vectors half the turned part apart: with that split both layouts load whole
// contiguous lines per warp.
#include <cuda_fp16.h>

#include "serving.cuh"

namespace dsa {
namespace {

constexpr int kRoThreads = 256;
constexpr int kRoTable = 2048;  // cosine pairs of a block (rotary_dim is at most 4096)

// The two 16-bit numbers of a word, and back (one rounding each).
template <typename T>
__device__ __forceinline__ float2 unpack(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <typename T>
__device__ __forceinline__ uint32_t pack(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float lo, float hi) { return pack_bf16x2(lo, hi); }
template <>
__device__ __forceinline__ uint32_t pack<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Two vectors of V elements of one head: 16 bytes each (V > 1), or one
// element each. turn() maps the pairs they hold: with the half layout a pair
// has an element in either; interleaved, each vector holds V / 2 pairs (with
// one element a vector the two are the pair).
template <typename T, int V>
struct Two {
  uint32_t a[4], d[4];
  __device__ __forceinline__ void load(const T* x, int o0, int o1, bool two) {
    const uint4 v = *reinterpret_cast<const uint4*>(x + o0);
    a[0] = v.x, a[1] = v.y, a[2] = v.z, a[3] = v.w;
    if (two) {
      const uint4 w = *reinterpret_cast<const uint4*>(x + o1);
      d[0] = w.x, d[1] = w.y, d[2] = w.z, d[3] = w.w;
    }
  }
  __device__ __forceinline__ void store(T* y, int o0, int o1, bool two) const {
    *reinterpret_cast<uint4*>(y + o0) = make_uint4(a[0], a[1], a[2], a[3]);
    if (two) *reinterpret_cast<uint4*>(y + o1) = make_uint4(d[0], d[1], d[2], d[3]);
  }
  template <bool kHalf>
  __device__ __forceinline__ void turn(const float2* cs) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 x0 = unpack<T>(a[k]), x1 = unpack<T>(d[k]);
        if constexpr (kHalf) {
          const float2 p0 = rotate_pair(x0.x, x1.x, cs[2 * k].x, cs[2 * k].y);
          const float2 p1 = rotate_pair(x0.y, x1.y, cs[2 * k + 1].x, cs[2 * k + 1].y);
          a[k] = pack<T>(p0.x, p1.x);
          d[k] = pack<T>(p0.y, p1.y);
        } else {
          const float2 p0 = rotate_pair(x0.x, x0.y, cs[k].x, cs[k].y);
          const float2 p1 = rotate_pair(x1.x, x1.y, cs[4 + k].x, cs[4 + k].y);
          a[k] = pack<T>(p0.x, p0.y);
          d[k] = pack<T>(p1.x, p1.y);
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; k += kHalf ? 1 : 2) {
        if constexpr (kHalf) {
          const float2 p0 = rotate_pair(__uint_as_float(a[k]), __uint_as_float(d[k]), cs[k].x, cs[k].y);
          a[k] = __float_as_uint(p0.x);
          d[k] = __float_as_uint(p0.y);
        } else {
          const float2 p0 = rotate_pair(__uint_as_float(a[k]), __uint_as_float(a[k + 1]), cs[k / 2].x, cs[k / 2].y);
          const float2 p1 = rotate_pair(__uint_as_float(d[k]), __uint_as_float(d[k + 1]), cs[2 + k / 2].x, cs[2 + k / 2].y);
          a[k] = __float_as_uint(p0.x), a[k + 1] = __float_as_uint(p0.y);
          d[k] = __float_as_uint(p1.x), d[k + 1] = __float_as_uint(p1.y);
        }
      }
    }
  }
};
template <typename T>
struct Two<T, 1> {
  T a, d;
  __device__ __forceinline__ void load(const T* x, int o0, int o1, bool two) {
    a = x[o0];
    if (two) d = x[o1];
  }
  __device__ __forceinline__ void store(T* y, int o0, int o1, bool two) const {
    y[o0] = a;
    if (two) y[o1] = d;
  }
  template <bool kHalf>
  __device__ __forceinline__ void turn(const float2* cs) {
    const float2 p = rotate_pair((float)a, (float)d, cs[0].x, cs[0].y);
    a = (T)p.x;
    d = (T)p.y;
  }
};

// Elements at which the two vectors of unit u start: a rotary unit's, or (from
// units_rot on) two of the copied vectors, of which the second may be missing.
template <int V, bool kHalf>
__device__ __forceinline__ void place(const RotaryParams& p, int u, int units_rot, int units, int* o0, int* o1, bool* two) {
  *two = true;
  if (u < units_rot) {
    *o0 = p.start + (V == 1 && !kHalf ? 2 * u : u * V);
    *o1 = V == 1 && !kHalf ? *o0 + 1 : *o0 + p.rotary_dim / 2;
  } else {
    const int vecs = (p.dim - p.rotary_dim) / V, first = p.start / V, skip = p.rotary_dim / V;
    const int c0 = u - units_rot, c1 = c0 + units - units_rot;
    *two = c1 < vecs;
    *o0 = (c0 + (c0 >= first ? skip : 0)) * V;
    *o1 = (c1 + (c1 >= first ? skip : 0)) * V;
  }
}
// The q-th of the V pairs of rotary unit u: with V > 1 and interleaved pairs,
// V / 2 in each of its two vectors, else one element in each.
template <int V, bool kHalf>
__device__ __forceinline__ int pair_of(const RotaryParams& p, int u, int q) {
  if (V == 1 || kHalf) return u * V + q;
  return q < V / 2 ? u * (V / 2) + q : p.rotary_dim / 4 + u * (V / 2) + q - V / 2;
}

// V: elements of a vector (16 bytes' worth, or 1 for sizes, strides or
// addresses that 16-byte accesses do not fit).
template <typename T, int V, bool kHalf>
__global__ void __launch_bounds__(kRoThreads) rotary_kernel(const RotaryParams p, int groups, int units_rot,
                                                            int units, int tokens_per_block) {
  extern __shared__ float2 table[];  // [tokens of the block][rotary_dim / 2], then turn fractions and positions
  const int per_token = groups * units;
  const int k = tokens_per_block > 1 ? (int)threadIdx.x / per_token : 0;
  const long long token = (long long)blockIdx.x * tokens_per_block + k;
  const int w = tokens_per_block > 1 ? (int)threadIdx.x - k * per_token : (int)(blockIdx.y * kRoThreads + threadIdx.x);
  const bool live = k < tokens_per_block && token < p.tokens && w < per_token;
  const int g = w / units, u = w - g * units;
  const uint32_t b = live ? (uint32_t)token / (uint32_t)p.queries : 0u;  // tokens < 2^31
  const uint32_t s = live ? (uint32_t)token - b * (uint32_t)p.queries : 0u;
  const T* x = static_cast<const T*>(p.x) + b * p.xs[0] + s * p.xs[1] + g * p.xs[2];
  T* y = static_cast<T*>(p.y) + b * p.ys[0] + s * p.ys[1] + g * p.ys[2];

  const bool turns = u < units_rot;
  int o0, o1;
  bool two;
  place<V, kHalf>(p, u, units_rot, units, &o0, &o1, &two);
  Two<T, V> cur;
  if (live) cur.load(x, o0, o1, two);

  const int pairs = p.rotary_dim / 2;
  unsigned long long* const fraction = reinterpret_cast<unsigned long long*>(table + tokens_per_block * pairs);
  long long* const position = reinterpret_cast<long long*>(fraction + pairs);
  for (int j = threadIdx.x; j < pairs; j += kRoThreads) fraction[j] = turn_fraction(__ldg(p.inv_freq + j));
  if (threadIdx.x < tokens_per_block) {  // at most kRoThreads
    const uint32_t t = (uint32_t)min((long long)blockIdx.x * tokens_per_block + threadIdx.x, p.tokens - 1);
    const uint32_t tb = t / (uint32_t)p.queries, ts = t - tb * (uint32_t)p.queries;
    const long long at = tb * p.ps[0] + ts * p.ps[1];
    position[threadIdx.x] = p.pos64 ? static_cast<const long long*>(p.positions)[at]
                                    : (long long)static_cast<const int32_t*>(p.positions)[at];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < tokens_per_block * pairs; i += kRoThreads) {
    const int tk = i / pairs, j = i - tk * pairs;
    rotary_cos_sin(position[tk], fraction[j], p.factor, p.sin_sign, &table[i].x, &table[i].y);
  }
  __syncthreads();
  if (!live) return;

  const long long xstep = groups * p.xs[2], ystep = groups * p.ys[2];
  float2 cs[V];
  if (turns) {
#pragma unroll
    for (int q = 0; q < V; ++q) cs[q] = table[k * pairs + pair_of<V, kHalf>(p, u, q)];
  }
  for (int h = g;;) {  // the next head's loads are under way while this one is turned
    Two<T, V> next;
    const bool more = (h += groups) < p.heads;
    if (more) next.load(x += xstep, o0, o1, two);
    if (turns) cur.template turn<kHalf>(cs);
    cur.store(y, o0, o1, two);
    if (!more) return;
    y += ystep;
    cur = next;
  }
}

// One head a token (k_rope, the indexer's keys): nobody shares a token's
// cosines, so a thread computes those of its pairs itself; the block keeps the
// pairs' turn fractions. Rotary units and copied ones are in different warps
// where they are many (cosines for half a warp cost as much as for a whole one).
// 65536 tokens, 64 wide: 6.3 us against 10.4 with the table; 128 wide with 64
// turned 8.8 against 13.9.
template <typename T, int V, bool kHalf>
__global__ void __launch_bounds__(kRoThreads, 4) rotary_rows_kernel(const RotaryParams p, int units_rot, int units,
                                                                    int tokens_per_block) {
  extern __shared__ unsigned long long fractions[];  // [rotary_dim / 2]
  const int tid = (int)threadIdx.x, rotary = tokens_per_block * units_rot;
  const bool turns = tid < rotary;
  const int mine = turns ? tid : tid - rotary, per_token = turns ? units_rot : units - units_rot;
  const int k = per_token > 0 ? mine / per_token : tokens_per_block;
  const int u = mine - k * per_token + (turns ? 0 : units_rot);
  const bool live = k < tokens_per_block;
  int o0 = 0, o1 = 0;
  bool two = false;
  if (live) place<V, kHalf>(p, u, units_rot, units, &o0, &o1, &two);
  const uint32_t stride = gridDim.x * (uint32_t)tokens_per_block, tokens = (uint32_t)p.tokens;  // < 2^31, stride < 2^20
  Two<T, V> cur;
  long long pos = 0;
  uint32_t b = 0, s = 0;
  auto load = [&](uint32_t t) {
    b = t / (uint32_t)p.queries;
    s = t - b * (uint32_t)p.queries;
    cur.load(static_cast<const T*>(p.x) + b * p.xs[0] + s * p.xs[1], o0, o1, two);
    if (turns) {
      const long long i = b * p.ps[0] + s * p.ps[1];
      pos = p.pos64 ? static_cast<const long long*>(p.positions)[i] : (long long)static_cast<const int32_t*>(p.positions)[i];
    }
  };
  uint32_t t = live ? blockIdx.x * (uint32_t)tokens_per_block + (uint32_t)k : tokens;
  if (t < tokens) load(t);
  for (int j = tid; j < p.rotary_dim / 2; j += kRoThreads) fractions[j] = turn_fraction(__ldg(p.inv_freq + j));
  __syncthreads();
  while (t < tokens) {
    if (turns) {
      float2 cs[V];
#pragma unroll
      for (int q = 0; q < V; ++q)
        rotary_cos_sin(pos, fractions[pair_of<V, kHalf>(p, u, q)], p.factor, p.sin_sign, &cs[q].x, &cs[q].y);
      cur.template turn<kHalf>(cs);
    }
    cur.store(static_cast<T*>(p.y) + b * p.ys[0] + s * p.ys[1], o0, o1, two);
    t += stride;
    if (t < tokens) load(t);
  }
}

template <typename T, int V>
cudaError_t launch_v(const RotaryParams& p, cudaStream_t stream) {
  const int units_rot = p.rotary_dim / (2 * V);
  const int copies = p.in_place ? 0 : (p.dim - p.rotary_dim) / V;
  const int units = units_rot + (copies + 1) / 2;
  if (p.heads == 1 && units <= kRoThreads) {
    const int per_block = kRoThreads / units;
    long long blocks = (p.tokens + per_block - 1) / per_block;
    if (blocks > 148 * 16) blocks = 148 * 16;
    const size_t smem = (size_t)(p.rotary_dim / 2) * sizeof(unsigned long long);
    if (p.half) rotary_rows_kernel<T, V, true><<<(unsigned)blocks, kRoThreads, smem, stream>>>(p, units_rot, units, per_block);
    else rotary_rows_kernel<T, V, false><<<(unsigned)blocks, kRoThreads, smem, stream>>>(p, units_rot, units, per_block);
    return cudaGetLastError();
  }
  // heads per thread: one while that leaves a part of the GPU idle, then as
  // many as keep it full (148 SMs x 2048 threads), so that a block's cosines
  // serve more rows. 4096 tokens x 64 heads x 128 (64 turned): 23.4 us, with
  // half as many threads 24.4, with four times as many 29.3.
  const long long want = 148LL * 2048;
  long long groups = (want + p.tokens * units - 1) / (p.tokens * units);
  if (groups > p.heads) groups = p.heads;
  while (groups & (groups - 1)) groups += groups & -groups;  // a power of two: whole lines per warp
  if (groups > p.heads) groups = p.heads;
  if (groups > 65535LL * kRoThreads / units) groups = 65535LL * kRoThreads / units;  // blocks of one token: grid.y
  const long long per_token = groups * units;
  int tpb = per_token < kRoThreads ? (int)(kRoThreads / per_token) : 1;
  if (tpb > kRoTable / (p.rotary_dim / 2)) tpb = kRoTable / (p.rotary_dim / 2);
  dim3 grid((unsigned)((p.tokens + tpb - 1) / tpb), 1, 1);
  if (tpb == 1) grid.y = (unsigned)((per_token + kRoThreads - 1) / kRoThreads);
  if (tpb < 1 || grid.y > 65535) return cudaErrorInvalidConfiguration;
  const size_t smem = (size_t)(tpb + 1) * (p.rotary_dim / 2) * sizeof(float2) + (size_t)tpb * sizeof(long long);
  if (p.half) rotary_kernel<T, V, true><<<grid, kRoThreads, smem, stream>>>(p, (int)groups, units_rot, units, tpb);
  else rotary_kernel<T, V, false><<<grid, kRoThreads, smem, stream>>>(p, (int)groups, units_rot, units, tpb);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_t(const RotaryParams& p, cudaStream_t stream) {
  constexpr int V = 16 / (int)sizeof(T);
  // 16-byte accesses: every vector of a row starts on a 16-byte boundary
  bool wide = p.rotary_dim % (2 * V) == 0 && p.start % V == 0 && (p.in_place || p.dim % V == 0);
  wide = wide && ((reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.y)) & 15u) == 0;
  for (int k = 0; k < 3; ++k) wide = wide && p.xs[k] % V == 0 && p.ys[k] % V == 0;
  return wide ? launch_v<T, V>(p, stream) : launch_v<T, 1>(p, stream);
}

}  // namespace

cudaError_t launch_rotary(const RotaryParams& p, int dtype, cudaStream_t stream) {
  switch (dtype) {
    case 0: return launch_t<__nv_bfloat16>(p, stream);
    case 1: return launch_t<__half>(p, stream);
    case 2: return launch_t<float>(p, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace dsa
