// Kernel parameters and launchers of the serving operators around the
// forward: rotary positions (rotary.cu), page plans (pages.cu) and cache
// appends (append.cu).
#pragma once

#include "dsa_common.cuh"

namespace dsa {

struct RotaryParams {
  const void* x;
  void* y;
  const void* positions;  // int32 or int64 [batch, queries]
  const double* inv_freq; // [rotary_dim / 2]
  long long xs[3], ys[3]; // strides in elements: batch, query, head
  long long ps[2];        // strides of positions
  long long tokens;       // batch * queries
  int queries, heads, dim, rotary_dim, start;
  int pos64, half, in_place;
  float factor;           // on cosines and sines
  float sin_sign;         // -1 for the inverse rotation
};
cudaError_t launch_rotary(const RotaryParams& p, int dtype, cudaStream_t stream);

struct PageParams {
  const int32_t* table_in;    // [batch, max_blocks]
  const int32_t* cached;      // [batch]
  const int32_t* new_lens;    // [batch]
  const int32_t* free_in;     // [num_blocks], a stack of free_count entries
  const int32_t* free_count;  // [1]
  const uint8_t* reset;       // [batch] or null
  int32_t* table_out;
  int32_t* seq_lens;          // [batch]
  int32_t* positions;         // [batch, queries]
  int32_t* lengths;           // [batch, queries]
  int32_t* slots;             // [batch, queries]
  int32_t* free_out;
  int32_t* free_count_out;
  int32_t* missing;           // [1]
  int4* rows;                 // workspace: [batch] {start, new tokens, pages kept, first page taken}
  int32_t* total;             // workspace: {stack height before the pages are taken, height without the returned pages}
  int batch, queries, max_blocks, num_blocks, block_size;
};
cudaError_t launch_plan_pages(const PageParams& p, cudaStream_t stream);

struct AppendParams {
  const __nv_bfloat16* kv;      // rows of 512
  const __nv_bfloat16* k_rope;  // rows of 64
  const int32_t* slots;         // [batch, queries]
  const int32_t* positions;     // [batch, queries] or null (k_rope is stored as given)
  const double* inv_freq;       // [32] or null
  __nv_bfloat16* kv_cache;      // [rows, 512] (BF16 cache)
  __nv_bfloat16* rope_cache;    // [rows, 64] (BF16 cache)
  uint8_t* cache;               // [rows, 656] (FP8 cache) or null
  long long kvs[2], krs[2];     // strides in elements: batch, query
  long long tokens, rows;
  int queries;                  // 0: token t lies at t * strides[1]
  int half;
  float factor;
};
cudaError_t launch_append_kv(const AppendParams& p, cudaStream_t stream);

#ifdef __CUDACC__
// freq / (2 pi), radians to turns a position, modulo one turn as a 64-bit
// fraction: positions are integers, so whole turns of the frequency do not
// matter, and position * fraction modulo 2^64 is the angle in turns, reduced
// exactly. 1 / (2 pi) and the product are taken in two FP64 pieces; the
// fraction is off by 2^-64 of a turn, the angle of position 2^31 by 2^-33.
__device__ __forceinline__ unsigned long long turn_fraction(double freq) {
  constexpr double kInvTwoPi = 0.15915494309189535, kInvTwoPiLo = -9.839338337591243e-18;
  const double hi = freq * kInvTwoPi;
  double lo = fma(freq, kInvTwoPi, -hi) + freq * kInvTwoPiLo;
  double t = hi - floor(hi);                      // exact
  // 2^32 t = whole + rest; the small piece joins the rest
  const double w = floor(t * 4294967296.0);
  lo = (t * 4294967296.0 - w) + lo * 4294967296.0;
  return ((unsigned long long)w << 32) + (unsigned long long)(long long)rint(lo * 4294967296.0);
}

// factor * (cos, sin) of position pos. The angle is position * fraction modulo
// one turn: three integer products, exact (an FP32 angle of position 10^6 would
// be off by up to 2^-5 radians). It is split into a quarter turn and
// x in [-1/8, 1/8] of a turn, whose sine and cosine are minimax polynomials
// (Remez exchange on sin(2 pi x) / x and (cos(2 pi x) - 1) / x^2 in x^2,
// errors 3.2e-9 relative and 5.4e-11): within 1.0e-7 after all roundings.
// ~25 instructions, where sincospif and FP64 reduction took ~90 and bound the
// rotation of single heads.
__device__ __forceinline__ void rotary_cos_sin(long long pos, unsigned long long fraction, float factor, float sin_sign,
                                               float* c, float* s) {
  const uint32_t turn = (uint32_t)(((unsigned long long)pos * fraction) >> 32);
  const uint32_t quarter = (turn + 0x20000000u) >> 30;
  const float x = (float)(int)(turn - (quarter << 30)) * 0x1p-32f;
  const float y = x * x;
  float sn = fmaf(y, -0x1.2d9302p+6f, 0x1.465e92p+6f);
  sn = fmaf(y, sn, -0x1.4abbbap+5f);
  sn = x * fmaf(y, sn, 0x1.921fb6p+2f);
  float cs = fmaf(y, 0x1.d9f7bcp+5f, -0x1.55c664p+6f);
  cs = fmaf(y, cs, 0x1.03c1dep+6f);
  cs = fmaf(y, cs, -0x1.3bd3ccp+4f);
  cs = fmaf(y, cs, 1.f);
  const float a = (quarter & 1u) ? sn : cs, b = (quarter & 1u) ? cs : sn;
  *c = __uint_as_float(__float_as_uint(a) ^ (((quarter + 1u) & 2u) << 30)) * factor;
  *s = __uint_as_float(__float_as_uint(b) ^ ((quarter & 2u) << 30)) * (factor * sin_sign);
}
// The turned pair, with the roundings spelled out: rotary and the cache
// appends give the same bits.
__device__ __forceinline__ float2 rotate_pair(float a, float b, float c, float s) {
  return make_float2(__fmaf_rn(a, c, -__fmul_rn(b, s)), __fmaf_rn(b, c, __fmul_rn(a, s)));
}
#endif

}  // namespace dsa
