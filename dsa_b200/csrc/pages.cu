// Page plan of one serving step: which pages the new tokens of every request
// take, the block tables, and where each token's cache row goes.
//
// For batch row b with c cached tokens (0 when `reset` gives the row to a new
// request), n new ones and pages of S tokens: the row keeps its first
// ceil(c / S) pages and takes ceil((c + n) / S) - ceil(c / S) from the top of
// the stack of free pages, rows in order; a reset row's old pages are pushed
// first. Token s of the row is at position c + s and in cache row
// table[(c + s) / S] * S + (c + s) % S. Without a page left an entry is -1,
// and so are the slots of its tokens.
//
// Two steps: the row step (one block, prefix sums over the rows, pushes) and
// the fill step (every table entry, token and stack entry on its own). Order
// is fixed by prefix sums, no atomics, so equal inputs give equal plans. The
// work is a few bytes per entry: latency bounds it, not bandwidth.
#include "serving.cuh"

namespace dsa {
namespace {

constexpr int kPgThreads = 1024;

// Exclusive sum of v over the block's threads; *sum gets the total.
__device__ __forceinline__ int block_exclusive(int v, int* warp_sums, int* sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += o;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int w = warp_sums[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) w += o;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  *sum = warp_sums[31];
  return x - v + (warp > 0 ? warp_sums[warp - 1] : 0);
}

__device__ __forceinline__ int pages_of(int tokens, int block_size) {
  return (int)(((long long)tokens + block_size - 1) / block_size);
}

__device__ void row_step(const PageParams& p) {
  __shared__ int warp_sums[32];
  __shared__ int had[kPgThreads];    // pages of a reset row (0: the row keeps its pages)
  __shared__ int count[kPgThreads];  // valid ones of them, then where they go on the stack
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int cap = p.max_blocks * p.block_size;
  const int free0 = min(max(*p.free_count, 0), p.num_blocks);
  int pushed = 0, taken = 0;
  for (int b0 = 0; b0 < p.batch; b0 += kPgThreads) {
    const int b = b0 + threadIdx.x;
    int start = 0, fresh = 0, kept = 0, need = 0, old = 0;
    if (b < p.batch) {
      const int cached = min(max(p.cached[b], 0), cap);
      const bool reset = p.reset != nullptr && p.reset[b] != 0;
      old = reset ? pages_of(cached, p.block_size) : 0;
      start = reset ? 0 : cached;
      fresh = min(min(max(p.new_lens[b], 0), p.queries), cap - start);
      kept = pages_of(start, p.block_size);
      need = pages_of(start + fresh, p.block_size) - kept;
    }
    if (p.reset != nullptr) {
      had[threadIdx.x] = old;
      count[threadIdx.x] = 0;
      __syncthreads();
      // a warp per reset row: how many of its entries name a page
      for (int r = warp; r < kPgThreads && b0 + r < p.batch; r += kPgThreads / 32) {
        if (had[r] == 0) continue;
        int n = 0;
        const int32_t* const row = p.table_in + (size_t)(b0 + r) * p.max_blocks;
        for (int j = lane; j < had[r]; j += 32) n += row[j] >= 0 && row[j] < p.num_blocks;
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) n += __shfl_xor_sync(0xffffffffu, n, d);
        if (lane == 0) count[r] = n;
      }
      __syncthreads();
      int sum;
      const int at = block_exclusive(count[threadIdx.x], warp_sums, &sum);
      __syncthreads();
      count[threadIdx.x] = at;
      __syncthreads();
      for (int r = warp; r < kPgThreads && b0 + r < p.batch; r += kPgThreads / 32) {
        if (had[r] == 0) continue;
        long long to = (long long)free0 + pushed + count[r];
        const int32_t* const row = p.table_in + (size_t)(b0 + r) * p.max_blocks;
        for (int j0 = 0; j0 < had[r]; j0 += 32) {
          const int e = j0 + lane < had[r] ? row[j0 + lane] : -1;
          const bool valid = e >= 0 && e < p.num_blocks;
          const uint32_t m = __ballot_sync(0xffffffffu, valid);
          const long long pos = to + __popc(m & ((1u << lane) - 1u));
          if (valid && pos < p.num_blocks) p.free_out[pos] = e;
          to += __popc(m);
        }
      }
      pushed += sum;
      __syncthreads();
    }
    int sum;
    const int at = block_exclusive(need, warp_sums, &sum);
    if (b < p.batch) {
      p.rows[b] = make_int4(start, fresh, kept, taken + at);
      p.seq_lens[b] = start + fresh;
    }
    taken += sum;
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const int total = (int)min((long long)free0 + pushed, (long long)p.num_blocks);
    p.total[0] = total;
    p.total[1] = free0;
    *p.free_count_out = max(total - taken, 0);
    *p.missing = max(taken - total, 0);
  }
}

// The a-th page taken from the stack of `total` pages: an entry below free0
// is the caller's, one above was pushed by the row step.
__device__ __forceinline__ int taken_page(const PageParams& p, int a, int total, int free0) {
  const int i = total - 1 - a;
  if (i < 0) return -1;
  return i < free0 ? p.free_in[i] : p.free_out[i];
}

__device__ void fill_step(const PageParams& p, long long first, long long stride) {
  const int total = p.total[0], free0 = p.total[1];
  const long long entries = (long long)p.batch * p.max_blocks;
  for (long long i = first; i < entries; i += stride) {
    const int b = (int)(i / p.max_blocks), j = (int)(i - (long long)b * p.max_blocks);
    const int4 r = p.rows[b];
    const int end = pages_of(r.x + r.y, p.block_size);
    if (j >= r.z && j < end) p.table_out[i] = taken_page(p, r.w + j - r.z, total, free0);
    else if (p.reset != nullptr && p.reset[b] != 0) p.table_out[i] = -1;
    else if (p.table_out != p.table_in) p.table_out[i] = p.table_in[i];
  }
  const long long tokens = (long long)p.batch * p.queries;
  for (long long i = first; i < tokens; i += stride) {
    const int b = (int)(i / p.queries), s = (int)(i - (long long)b * p.queries);
    const int4 r = p.rows[b];
    int pos = -1, slot = -1;
    if (s < r.y) {
      pos = r.x + s;
      const int j = pos / p.block_size;
      // pages that the row keeps are not written by this step
      const int page = j < r.z ? p.table_in[(size_t)b * p.max_blocks + j] : taken_page(p, r.w + j - r.z, total, free0);
      if (page >= 0 && page < p.num_blocks) slot = page * p.block_size + pos % p.block_size;
    }
    p.positions[i] = pos;
    p.lengths[i] = pos + 1;
    p.slots[i] = slot;
  }
  if (p.free_out != p.free_in)
    for (long long i = first; i < p.num_blocks; i += stride)
      if (i < free0 || i >= total) p.free_out[i] = p.free_in[i];
}

__global__ void __launch_bounds__(kPgThreads) plan_rows_kernel(const PageParams p) { row_step(p); }

__global__ void __launch_bounds__(256) plan_fill_kernel(const PageParams p) {
  fill_step(p, (long long)blockIdx.x * 256 + threadIdx.x, (long long)gridDim.x * 256);
}

}  // namespace

cudaError_t launch_plan_pages(const PageParams& p, cudaStream_t stream) {
  plan_rows_kernel<<<1, kPgThreads, 0, stream>>>(p);
  const long long work = (long long)p.batch * (p.max_blocks > p.queries ? p.max_blocks : p.queries);
  long long most = work > p.num_blocks ? work : p.num_blocks;
  long long blocks = (most + 255) / 256;
  if (blocks > 148 * 8) blocks = 148 * 8;
  plan_fill_kernel<<<(unsigned)blocks, 256, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace dsa
