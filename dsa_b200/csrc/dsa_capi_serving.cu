// extern "C" boundary of the serving operators (declared in
// include/dsa_b200.h): what the C ABI can see is checked here (null pointers,
// sizes, alignment), shapes and dtypes in the Python mirrors
// (dsa_b200/rope.py, dsa_b200/paging.py).
#include <cuda_runtime.h>

#include <cmath>
#include <cstring>

#include "../../include/dsa_b200.h"
#include "serving.cuh"

namespace {

constexpr int64_t kMaxInt = 0x7fffffffLL;

bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1u)) == 0; }

// a * b <= limit for positive a, b, without overflow
bool product_ok(int64_t a, int64_t b, int64_t limit = kMaxInt) { return a > 0 && b > 0 && a <= limit / b; }

int launch_status(cudaError_t err) { return err == cudaSuccess ? DSA_STATUS_OK : DSA_STATUS_LAUNCH_FAILED; }

bool plan_ok(const dsa_plan_pages_args_t* a) {
  return a != nullptr && product_ok(a->batch, a->queries) && product_ok(a->batch, a->max_blocks) &&
         product_ok(a->max_blocks, a->block_size) && product_ok(a->num_blocks, a->block_size);
}

}  // namespace

extern "C" {

int dsa_rotary(const dsa_rotary_args_t* a, void* stream) {
  if (a == nullptr || !a->x || !a->y || !a->positions || !a->inv_freq) return DSA_STATUS_BAD_ARGUMENT;
  if (!product_ok(a->batch, a->queries) || a->heads <= 0 || a->heads > kMaxInt || a->dim <= 0 || a->dim > 65536)
    return DSA_STATUS_BAD_ARGUMENT;
  if (a->rotary_dim <= 0 || a->rotary_dim % 2 != 0 || a->start < 0 || a->start > a->dim - a->rotary_dim)
    return DSA_STATUS_BAD_ARGUMENT;
  if (a->dtype < DSA_BF16 || a->dtype > DSA_FP32 || (a->layout != DSA_ROPE_INTERLEAVED && a->layout != DSA_ROPE_HALF))
    return DSA_STATUS_BAD_ARGUMENT;
  const unsigned item = a->dtype == DSA_FP32 ? 4u : 2u;
  if (!aligned(a->x, item) || !aligned(a->y, item) || !aligned(a->inv_freq, 8) ||
      !aligned(a->positions, a->positions64 ? 8 : 4))
    return DSA_STATUS_BAD_ARGUMENT;
  if (!std::isfinite(a->attention_factor)) return DSA_STATUS_BAD_ARGUMENT;
  dsa::RotaryParams p;
  p.x = a->x;
  p.y = a->y;
  p.positions = a->positions;
  p.inv_freq = a->inv_freq;
  // the stride of a dimension of one element is never walked
  const int64_t sizes[3] = {a->batch, a->queries, a->heads};
  p.in_place = a->x == a->y;
  for (int k = 0; k < 3; ++k) {
    p.xs[k] = sizes[k] > 1 ? a->x_stride[k] : 0;
    p.ys[k] = sizes[k] > 1 ? a->y_stride[k] : 0;
    if (p.in_place && p.xs[k] != p.ys[k]) return DSA_STATUS_BAD_ARGUMENT;
    if (k < 2) p.ps[k] = sizes[k] > 1 ? a->position_stride[k] : 0;
  }
  p.tokens = a->batch * a->queries;
  p.queries = (int)a->queries;
  p.heads = (int)a->heads;
  p.dim = (int)a->dim;
  p.rotary_dim = a->rotary_dim;
  p.start = a->start;
  p.pos64 = a->positions64 != 0;
  p.half = a->layout == DSA_ROPE_HALF;
  p.factor = a->attention_factor;
  p.sin_sign = a->inverse ? -1.f : 1.f;
  return launch_status(dsa::launch_rotary(p, a->dtype, static_cast<cudaStream_t>(stream)));
}

uint64_t dsa_plan_pages_workspace_bytes(const dsa_plan_pages_args_t* a) {
  return plan_ok(a) ? (uint64_t)a->batch * sizeof(int4) + 16u : 0;
}

int dsa_plan_pages(const dsa_plan_pages_args_t* a, void* stream) {
  if (!plan_ok(a)) return DSA_STATUS_BAD_ARGUMENT;
  const void* const need[] = {a->block_table, a->cached_lens, a->new_lens, a->free_blocks, a->free_count,
                              a->table_out, a->seq_lens, a->positions, a->lengths, a->slots, a->free_blocks_out,
                              a->free_count_out, a->missing};
  for (const void* q : need)
    if (q == nullptr || !aligned(q, 4)) return DSA_STATUS_BAD_ARGUMENT;
  if (a->workspace == nullptr || a->workspace_bytes < dsa_plan_pages_workspace_bytes(a) || !aligned(a->workspace, 16))
    return DSA_STATUS_WORKSPACE_TOO_SMALL;
  dsa::PageParams p;
  p.table_in = a->block_table;
  p.cached = a->cached_lens;
  p.new_lens = a->new_lens;
  p.free_in = a->free_blocks;
  p.free_count = a->free_count;
  p.reset = a->reset;
  p.table_out = a->table_out;
  p.seq_lens = a->seq_lens;
  p.positions = a->positions;
  p.lengths = a->lengths;
  p.slots = a->slots;
  p.free_out = a->free_blocks_out;
  p.free_count_out = a->free_count_out;
  p.missing = a->missing;
  p.total = static_cast<int32_t*>(a->workspace);
  p.rows = reinterpret_cast<int4*>(static_cast<char*>(a->workspace) + 16);
  p.batch = (int)a->batch;
  p.queries = (int)a->queries;
  p.max_blocks = (int)a->max_blocks;
  p.num_blocks = (int)a->num_blocks;
  p.block_size = (int)a->block_size;
  return launch_status(dsa::launch_plan_pages(p, static_cast<cudaStream_t>(stream)));
}

int dsa_append_kv(const dsa_append_kv_args_t* a, void* stream) {
  if (a == nullptr || !a->kv || !a->k_rope || !a->slots) return DSA_STATUS_BAD_ARGUMENT;
  if (!product_ok(a->batch, a->queries) || a->rows <= 0 || a->rows > kMaxInt) return DSA_STATUS_BAD_ARGUMENT;
  if (a->cache != nullptr ? (a->kv_cache != nullptr || a->k_rope_cache != nullptr || !aligned(a->cache, 16))
                          : (!a->kv_cache || !a->k_rope_cache || !aligned(a->kv_cache, 16) || !aligned(a->k_rope_cache, 16)))
    return DSA_STATUS_BAD_ARGUMENT;
  if ((a->inv_freq != nullptr) != (a->positions != nullptr)) return DSA_STATUS_BAD_ARGUMENT;
  if (a->layout != DSA_ROPE_INTERLEAVED && a->layout != DSA_ROPE_HALF) return DSA_STATUS_BAD_ARGUMENT;
  if (!aligned(a->kv, 2) || !aligned(a->k_rope, 2) || !aligned(a->slots, 4) || !aligned(a->inv_freq, 8) ||
      !aligned(a->positions, 4) || !std::isfinite(a->attention_factor))
    return DSA_STATUS_BAD_ARGUMENT;
  dsa::AppendParams p;
  p.kv = static_cast<const __nv_bfloat16*>(a->kv);
  p.k_rope = static_cast<const __nv_bfloat16*>(a->k_rope);
  p.slots = a->slots;
  p.positions = a->positions;
  p.inv_freq = a->inv_freq;
  p.kv_cache = static_cast<__nv_bfloat16*>(a->kv_cache);
  p.rope_cache = static_cast<__nv_bfloat16*>(a->k_rope_cache);
  p.cache = static_cast<uint8_t*>(a->cache);
  for (int k = 0; k < 2; ++k) {
    const bool walked = (k == 0 ? a->batch : a->queries) > 1;
    p.kvs[k] = walked ? a->kv_stride[k] : 0;
    p.krs[k] = walked ? a->k_rope_stride[k] : 0;
  }
  p.tokens = a->batch * a->queries;
  p.rows = a->rows;
  p.queries = (int)a->queries;
  p.half = a->layout == DSA_ROPE_HALF;
  p.factor = a->attention_factor;
  return launch_status(dsa::launch_append_kv(p, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
