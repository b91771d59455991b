// Rotary positions: y = x with `rotary_dim` of its `dim` elements turned by
// the token's position,
//   y_a = f (x_a cos t - x_b sin t),  y_b = f (x_b cos t + x_a sin t),
//   t = position * inv_freq[i],  f = the attention factor,
// over the pairs (a, b) = (2i, 2i + 1) (interleaved) or (i, i + rotary_dim/2)
// (half). The other elements are copied. The gradient of y with respect to x
// is the same map with -t, so the backward pass is this kernel again.
//
// Bound: HBM, 2 * dim elements per head row. The cosines cost ~40 FP32 and 5
// FP64 instructions a pair, more than the memory time of one row, and depend
// on the token alone: a thread owns fixed pairs of one token and walks over
// heads h, h + groups, ..., so they are computed once per thread and stay in
// registers. A unit is two 16-byte vectors half the turned part apart: with
// that split both layouts load whole contiguous lines per warp.
#include <cuda_fp16.h>

#include "serving.cuh"

namespace dsa {
namespace {

constexpr int kRoThreads = 256;

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(float v) { return v; }
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }

// V elements of T loaded and stored as one access.
template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T e[V];
};

// V: elements of a vector (16 bytes' worth, or 1 for sizes, strides or
// addresses that 16-byte accesses do not fit).
template <typename T, int V>
__global__ void __launch_bounds__(kRoThreads) rotary_kernel(const RotaryParams p, int groups, int units_rot,
                                                            int units, int tokens_per_block) {
  using VT = Vec<T, V>;
  const int per_token = groups * units;
  long long token;
  int w;
  if (tokens_per_block > 1) {
    const int k = threadIdx.x / per_token;
    if (k >= tokens_per_block) return;
    token = (long long)blockIdx.x * tokens_per_block + k;
    w = threadIdx.x - k * per_token;
  } else {
    token = blockIdx.x;
    w = blockIdx.y * kRoThreads + threadIdx.x;
  }
  if (token >= p.tokens || w >= per_token) return;
  const int g = w / units, u = w - g * units;
  const int b = (int)(token / p.queries), s = (int)(token - (long long)b * p.queries);
  const T* const x = static_cast<const T*>(p.x) + b * p.xs[0] + s * p.xs[1];
  T* const y = static_cast<T*>(p.y) + b * p.ys[0] + s * p.ys[1];

  if (u >= units_rot) {  // copied elements: vectors c and c + units_copy
    const int vecs = (p.dim - p.rotary_dim) / V, first = p.start / V, units_copy = units - units_rot;
    int c0 = u - units_rot, c1 = c0 + units_copy;
    const bool two = c1 < vecs;
    const int skip = p.rotary_dim / V;
    c0 += c0 >= first ? skip : 0;
    c1 += c1 >= first ? skip : 0;
#pragma unroll 4
    for (int h = g; h < p.heads; h += groups) {
      const T* const xh = x + h * p.xs[2];
      T* const yh = y + h * p.ys[2];
      const VT v0 = *reinterpret_cast<const VT*>(xh + c0 * V);
      if (two) *reinterpret_cast<VT*>(yh + c1 * V) = *reinterpret_cast<const VT*>(xh + c1 * V);
      *reinterpret_cast<VT*>(yh + c0 * V) = v0;
    }
    return;
  }

  // this thread's V pairs: with V > 1 and interleaved pairs, V / 2 in each of
  // its two vectors
  const long long pos = p.pos64 ? static_cast<const long long*>(p.positions)[b * p.ps[0] + s * p.ps[1]]
                                : (long long)static_cast<const int32_t*>(p.positions)[b * p.ps[0] + s * p.ps[1]];
  const int o0 = p.start + (V == 1 && !p.half ? 2 * u : u * V);
  const int o1 = V == 1 && !p.half ? o0 + 1 : o0 + p.rotary_dim / 2;
  float c[V], sn[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    int i = u * V + k;
    if (V > 1 && !p.half) i = k < V / 2 ? u * (V / 2) + k : p.rotary_dim / 4 + u * (V / 2) + k - V / 2;
    rotary_cos_sin(pos, __ldg(p.inv_freq + i), p.factor, p.sin_sign, &c[k], &sn[k]);
  }
  const bool across = V == 1 || p.half;  // a pair's elements are in different vectors
#pragma unroll 4
  for (int h = g; h < p.heads; h += groups) {
    const VT a = *reinterpret_cast<const VT*>(x + h * p.xs[2] + o0);
    const VT d = *reinterpret_cast<const VT*>(x + h * p.xs[2] + o1);
    VT ra, rd;
    if (across) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float2 t = rotate_pair(to_f(a.e[k]), to_f(d.e[k]), c[k], sn[k]);
        ra.e[k] = from_f<T>(t.x);
        rd.e[k] = from_f<T>(t.y);
      }
    } else {
#pragma unroll
      for (int k = 0; k < V / 2; ++k) {
        const float2 t = rotate_pair(to_f(a.e[2 * k]), to_f(a.e[2 * k + 1]), c[k], sn[k]);
        const float2 v = rotate_pair(to_f(d.e[2 * k]), to_f(d.e[2 * k + 1]), c[k + V / 2], sn[k + V / 2]);
        ra.e[2 * k] = from_f<T>(t.x);
        ra.e[2 * k + 1] = from_f<T>(t.y);
        rd.e[2 * k] = from_f<T>(v.x);
        rd.e[2 * k + 1] = from_f<T>(v.y);
      }
    }
    *reinterpret_cast<VT*>(y + h * p.ys[2] + o0) = ra;
    *reinterpret_cast<VT*>(y + h * p.ys[2] + o1) = rd;
  }
}

template <typename T, int V>
cudaError_t launch_v(const RotaryParams& p, cudaStream_t stream) {
  const int units_rot = p.rotary_dim / (2 * V);
  const int copies = p.in_place ? 0 : (p.dim - p.rotary_dim) / V;
  const int units = units_rot + (copies + 1) / 2;
  // heads per thread: one while that leaves a part of the GPU idle (148 SMs
  // x 2048 threads), then as many as keep the GPU full, so that a thread's
  // cosines serve more rows
  const long long want = 148LL * 2048;
  long long groups = (want + p.tokens * units - 1) / (p.tokens * units);
  if (groups > p.heads) groups = p.heads;
  while (groups & (groups - 1)) groups += groups & -groups;  // a power of two: whole lines per warp
  if (groups > p.heads) groups = p.heads;
  const long long per_token = groups * units;
  if (per_token > 0x7fffffffLL / 2) return cudaErrorInvalidConfiguration;
  int tpb = per_token < kRoThreads ? (int)(kRoThreads / per_token) : 1;
  dim3 grid((unsigned)((p.tokens + tpb - 1) / tpb), 1, 1);
  if (tpb == 1) grid.y = (unsigned)((per_token + kRoThreads - 1) / kRoThreads);
  if (grid.y > 65535) return cudaErrorInvalidConfiguration;
  rotary_kernel<T, V><<<grid, kRoThreads, 0, stream>>>(p, (int)groups, units_rot, units, tpb);
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
