// extern "C" boundary of the serving operators (declared in
// include/dsa_b200.h): what the C ABI can see is checked here (null pointers,
// sizes, alignment), shapes and dtypes in the Python mirrors
// (dsa_b200/rope.py, dsa_b200/paging.py, dsa_b200/shared_prefix.py).
#include <cuda_runtime.h>

#include <cmath>
#include <cstring>

#include "../../include/dsa_b200.h"
#include "prefix.cuh"
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

constexpr uint64_t kAlign = 256;
uint64_t align_up(uint64_t x) { return (x + kAlign - 1) / kAlign * kAlign; }

// Launches of one shared-prefix call and its workspace.
struct PrefixPlan {
  int64_t tokens, rows, row_tiles;
  int group, split, own_split;  // own_split 0: no own keys
  bool direct;           // the prefix kernel writes the output
  uint64_t num, max, sum, own_num, own_max, own_sum, total;
};

// Row tiles per item (1 or 2) and key splits of the prefix: a cluster's time
// is its tiles plus a start and an end of about twelve (launch, TMEM, Q, first
// loads, stores), in waves of the resident clusters; split partials cost a write
// and a read of 2 KB a row, about 5 TB/s, and the join ~0.3 us a part (96 rows
// over 1000 keys: 8 splits 17.9 us, 16 splits 20.6). A tile of 64 keys takes a cluster of one row tile ~1,400
// cycles and one of two ~1,200; the latter leaves half a cluster idle when the
// row tiles are odd. A lone row tile takes two all the same (half of the cluster
// works on a repeated row): 16 rows over 1,000 keys 15.6 us against 16.2 with
// one, 128 rows 18.9 against 19.5, 128 rows over 32,768 keys 41.3 against 40.4.
// The keys counted are the buffer's: how many of them are in use is known on the
// device alone.
struct PrefixEstimate {
  double us, kernel_us;  // with and without what the partials cost afterwards
  int split;
  int64_t sms;           // that hold a CTA of the kernel
};
PrefixEstimate prefix_split(int64_t row_tiles, int64_t keys, int group) {
  int clusters = dsa::prefix_max_clusters(group);
  if (clusters <= 0) clusters = 74 / group;
  const int64_t tiles = (keys + 63) / 64, sets = (row_tiles + group - 1) / group;
  const double tile_us = group == 1 ? 0.85 : 0.73;
  PrefixEstimate best{0, 0, 1, 0};
  // more than four waves of items never pay
  for (int s = 1; s <= 128 && s <= tiles && (s == 1 || sets * s <= 4 * (int64_t)clusters); ++s) {
    const int64_t waves = (sets * s + clusters - 1) / clusters;
    const double kernel = tile_us * (double)waves * (double)((tiles + s - 1) / s + 12);
    const double us = kernel + (s > 1 ? 1.0 + 0.3 * s + (double)row_tiles * s * 128 * 4096 / 5e6 : 0.0);
    if (s == 1 || us < best.us) best = {us, kernel, s, 2 * group * (sets * s < clusters ? sets * s : (int64_t)clusters)};
  }
  return best;
}

// Splits of the own keys, which run beside the prefix kernel: `idle` places
// (CTAs or pairs) are free from the start, `busy` ones once that kernel ends,
// and items of one length d go to whichever is free, so what counts is how many
// rounds remain when the prefix is done. The end is the first time by which the
// places have run all items; each split adds its partials. A kernel time 5 %
// off either way counts as likely, so that a choice does not hang on an item
// that just fits. Times in us, fitted to thirteen (stream) and ten (pair)
// shapes, within 1.5 % of the best split on average. Against one wave of splits
// for all places: 64 queries x 16 heads, 32768 + 2048 keys 107 -> 102; 200 x 16,
// 4096 + 2048 177 -> 144; 8 x 128, 32768 + 2048 103 -> 70 (all of them beside).
int own_splits(int64_t items, int64_t rows, int64_t tiles, bool pair, int64_t idle, int64_t busy, double prefix_us) {
  const double item_us = pair ? 9.5 : 6, tile_us = pair ? 0.88 : 1.8, late_us = pair ? 2 : 10;
  const double part_us = (pair ? 0.2 : 0.5) + (double)rows * 4096 / (pair ? 2.5e6 : 5e6);
  int split = 1;
  double best = 0;
  for (int s = 1; s <= 16 && (s == 1 || s <= tiles / 2); ++s) {
    const double d = item_us + tile_us * (double)((tiles + s - 1) / s), n = (double)items * s;
    double us = part_us * s;
    for (const double f : {0.95, 1.0, 1.05}) {
      const double t0 = prefix_us * f + late_us;
      const auto done = [&](double t) {
        return (double)idle * std::floor(t / d + 1e-6) + (t < t0 ? 0.0 : (double)busy * std::floor((t - t0) / d + 1e-6));
      };
      // places that never pause would be through by `low`; an item ends at a multiple of d
      const double alone = idle > 0 ? n * d / (double)idle : t0 + 1;
      const double low = alone <= t0 ? alone : (n * d + (double)busy * t0) / (double)(idle + busy);
      double end = 1e300;
      for (const double from : {0.0, t0}) {
        double k = std::fmax(0.0, std::floor((low - from) / d));
        while (done(from + k * d) < n) k += 1;
        end = std::fmin(end, from + k * d);
      }
      us += std::fmax(end, t0) / 3;
    }
    if (s == 1 || us < best) {
      best = us;
      split = s;
    }
  }
  return split;
}

bool plan_prefix(const dsa_fwd_args_t* a, const dsa_prefix_kv_t* px, PrefixPlan* plan) {
  if (a == nullptr || px == nullptr || a->launch.family != DSA_FAMILY_AUTO) return false;
  if (!product_ok(a->batch, a->queries) || a->heads <= 0 || a->heads > 65536 || a->heads % 16 != 0) return false;
  if (px->rows <= 0 || px->rows > (1LL << 26)) return false;
  const bool own = a->topk > 0;
  if (a->topk < 0 || a->topk > kMaxInt || (own && (!product_ok(a->batch, a->length)))) return false;
  plan->tokens = a->batch * a->queries;
  if (!product_ok(plan->tokens, a->heads, 1LL << 37)) return false;
  plan->rows = plan->tokens * a->heads;
  plan->row_tiles = (plan->rows + 127) / 128;
  const PrefixEstimate one = prefix_split(plan->row_tiles, px->rows, 1), two = prefix_split(plan->row_tiles, px->rows, 2);
  const PrefixEstimate& taken = two.us < one.us ? two : one;
  plan->group = two.us < one.us ? 2 : 1;
  plan->split = taken.split;
  if ((plan->row_tiles + 1) * plan->split > kMaxInt / 2) return false;
  plan->own_split = 0;
  if (own) {
    // own keys: pairs of CTAs (H = 128) or the stream family's CTAs, a 16-head group each
    const bool pair = a->heads == 128;
    int64_t places = pair ? dsa::pair_max_ctas() / 2 : dsa::stream_max_ctas();
    if (places <= 0) places = pair ? 74 : 296;
    const int64_t sms = 148, busy = places * (taken.sms < sms ? taken.sms : sms) / sms;
    plan->own_split = own_splits(pair ? plan->tokens : plan->tokens * (a->heads / 16), plan->rows, (a->topk + 31) / 32, pair,
                                 places - busy, busy, taken.kernel_us);
  }
  plan->direct = !own && plan->split == 1;
  plan->num = plan->max = plan->sum = plan->own_num = plan->own_max = plan->own_sum = plan->total = 0;
  if (plan->direct) return true;
  const uint64_t parts = (uint64_t)plan->row_tiles * (uint64_t)plan->split * 128u;
  plan->max = align_up(parts * dsa::kDimLatent * 4u);
  plan->sum = plan->max + align_up(parts * 4u);
  plan->total = plan->own_num = plan->sum + align_up(parts * 4u);
  if (own) {
    const uint64_t mine = (uint64_t)plan->rows * (uint64_t)plan->own_split;
    plan->own_max = plan->own_num + align_up(mine * dsa::kDimLatent * 4u);
    plan->own_sum = plan->own_max + align_up(mine * 4u);
    plan->total = plan->own_sum + align_up(mine * 4u);
  }
  return true;
}

}  // namespace

extern "C" {

int dsa_rotary(const dsa_rotary_args_t* a, void* stream) {
  if (a == nullptr || !a->x || !a->y || !a->positions || !a->inv_freq) return DSA_STATUS_BAD_ARGUMENT;
  if (!product_ok(a->batch, a->queries) || a->heads <= 0 || a->heads > kMaxInt || a->dim <= 0 || a->dim > 65536)
    return DSA_STATUS_BAD_ARGUMENT;
  if (a->rotary_dim <= 0 || a->rotary_dim > 4096 || a->rotary_dim % 2 != 0 || a->start < 0 || a->start > a->dim - a->rotary_dim)
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
  // tokens that one stride walks over need no division by the queries
  p.queries = (int)a->queries;
  if (a->queries == 1) {
    p.kvs[1] = p.kvs[0];
    p.krs[1] = p.krs[0];
    p.queries = 0;
  } else if (a->batch == 1 || (p.kvs[0] == a->queries * p.kvs[1] && p.krs[0] == a->queries * p.krs[1])) {
    p.queries = 0;
  }
  p.half = a->layout == DSA_ROPE_HALF;
  p.factor = a->attention_factor;
  return launch_status(dsa::launch_append_kv(p, static_cast<cudaStream_t>(stream)));
}

uint64_t dsa_fwd_prefix_workspace_bytes(const dsa_fwd_args_t* a, const dsa_prefix_kv_t* px) {
  PrefixPlan plan;
  return plan_prefix(a, px, &plan) ? plan.total : 0;
}

int dsa_fwd_prefix_plan(const dsa_fwd_args_t* a, const dsa_prefix_kv_t* px, int32_t out[3]) {
  PrefixPlan plan;
  if (out == nullptr || !plan_prefix(a, px, &plan)) return DSA_STATUS_BAD_ARGUMENT;
  out[0] = plan.group;
  out[1] = plan.split;
  out[2] = plan.own_split;
  return DSA_STATUS_OK;
}

int dsa_sparse_mla_fwd_prefix(const dsa_fwd_args_t* a, const dsa_prefix_kv_t* px, void* stream) {
  PrefixPlan plan;
  if (!plan_prefix(a, px, &plan)) return DSA_STATUS_BAD_ARGUMENT;
  const bool own = a->topk > 0;
  if (!a->q || !a->q_rope || !a->output || !a->softmax_max || !a->softmax_sum || !px->kv || !px->k_rope)
    return DSA_STATUS_BAD_ARGUMENT;
  if (own != (a->kv != nullptr) || own != (a->k_rope != nullptr) || own != (a->indices != nullptr))
    return DSA_STATUS_BAD_ARGUMENT;
  if (!aligned(a->q, 16) || !aligned(a->q_rope, 16) || !aligned(a->output, 16) || !aligned(px->kv, 16) ||
      !aligned(px->k_rope, 16) || !aligned(a->kv, 16) || !aligned(a->k_rope, 16) || !aligned(px->length, 4))
    return DSA_STATUS_BAD_ARGUMENT;
  if (plan.total > 0 && (a->workspace == nullptr || a->workspace_bytes < plan.total || !aligned(a->workspace, kAlign)))
    return DSA_STATUS_WORKSPACE_TOO_SMALL;
  char* const ws = static_cast<char*>(a->workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);

  dsa::FwdParams f;
  std::memset(&f, 0, sizeof(f));
  if (!dsa::fill_scale(a->scale, f)) return DSA_STATUS_BAD_ARGUMENT;
  dsa::PrefixParams p;
  p.q = static_cast<const __nv_bfloat16*>(a->q);
  p.q_rope = static_cast<const __nv_bfloat16*>(a->q_rope);
  p.length = px->length;
  p.out = static_cast<__nv_bfloat16*>(a->output);
  p.out_max = a->softmax_max;
  p.out_sum = a->softmax_sum;
  p.part_num = plan.direct ? nullptr : reinterpret_cast<float*>(ws + plan.num);
  p.part_max = reinterpret_cast<float*>(ws + plan.max);
  p.part_sum = reinterpret_cast<float*>(ws + plan.sum);
  p.status = a->status;
  p.rows = plan.rows;
  p.keys = (int)px->rows;
  p.split = plan.split;
  p.group = plan.group;
  p.scale_div = f.scale_div;
  p.scale_log2 = f.scale_log2;
  int st = launch_status(dsa::launch_fwd_prefix(p, px->kv, px->k_rope, s));
  if (st != DSA_STATUS_OK || plan.direct) return st;

  dsa::JoinParams j;
  j.part_num = p.part_num;
  j.part_max = p.part_max;
  j.part_sum = p.part_sum;
  j.own_num = reinterpret_cast<float*>(ws + plan.own_num);
  j.own_max = reinterpret_cast<float*>(ws + plan.own_max);
  j.own_sum = reinterpret_cast<float*>(ws + plan.own_sum);
  j.out = p.out;
  j.out_max = p.out_max;
  j.out_sum = p.out_sum;
  j.rows = plan.rows;
  j.heads = (int)a->heads;
  j.split = plan.split;
  j.own_split = plan.own_split;
  if (own) {
    f.q = p.q;
    f.q_rope = p.q_rope;
    f.kv = static_cast<const __nv_bfloat16*>(a->kv);
    f.k_rope = static_cast<const __nv_bfloat16*>(a->k_rope);
    f.ids = a->indices;
    f.part_num = reinterpret_cast<float*>(ws + plan.own_num);
    f.part_max = reinterpret_cast<float*>(ws + plan.own_max);
    f.part_sum = reinterpret_cast<float*>(ws + plan.own_sum);
    f.status = a->status;
    f.batch = (int)a->batch;
    f.queries = (int)a->queries;
    f.heads = (int)a->heads;
    f.length = (int)a->length;
    f.topk = (int)a->topk;
    f.tokens = (int)plan.tokens;
    f.split = plan.own_split;
    f.keys_per_tile = 32;
    f.heads_per_cta = a->heads == 128 ? 128 : 16;
    f.beside_previous = 1;  // fills the SMs that the prefix kernel leaves
    st = launch_status(a->heads == 128 ? dsa::launch_fwd_pair(f, s) : dsa::launch_fwd_stream(f, s));
    if (st != DSA_STATUS_OK) return st;
  }
  return launch_status(dsa::launch_prefix_join(j, s));
}

}  // extern "C"
