// Page plan of one serving step: which pages the new tokens of every request
// take, the block tables, and where each token's cache row goes.
//
// For batch row b with c cached tokens (0 when `reset` gives the row to a new
// request), n new ones and pages of S tokens: the row keeps its first
// ceil(c / S) pages and takes ceil((c + n) / S) - ceil(c / S) from the top of
// the stack of free pages, rows in order; a reset row's old pages are pushed
// first. Token s of the row is at position c + s and in cache row
// table[(c + s) / S] * S + (c + s) % S. Without a page left an entry is -1,
// and so are the slots of its tokens. Such a page stays missing: what its
// earlier tokens were to hold is lost, and a page given to the entry later would
// show a former owner's rows in their place. Steps that go on in it count it again.
//
// Two steps: the row step (one block, prefix sums over the rows, pushes) and
// the fill step (every table entry, token and stack entry on its own). Order
// is fixed by prefix sums, so equal inputs give equal plans. The work is a few
// bytes per entry: latency bounds it, not bandwidth. They are two launches, the
// second a programmatic one, which waits for the first on the GPU (the row step
// lets it start only at its own end); one launch of an eight-block cluster with
// its barrier between the steps was no faster for small plans (6.2 us) and
// slower for others (64 rows of 1024 pages 11.8 against 9.3 us).
#include "serving.cuh"

namespace dsa {
namespace {

constexpr int kPgThreads = 1024;
constexpr int kPgAhead = 4;  // loads of a returned row in flight

// Exclusive sums of v.x and v.y over the block's threads; *sum gets the totals.
__device__ __forceinline__ int2 block_exclusive(int2 v, int2* warp_sums, int2* sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto inclusive = [&](int2 x) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int ox = __shfl_up_sync(0xffffffffu, x.x, d), oy = __shfl_up_sync(0xffffffffu, x.y, d);
      if (lane >= d) x.x += ox, x.y += oy;
    }
    return x;
  };
  const int2 x = inclusive(v);
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  const int2 w = inclusive(warp_sums[lane]);  // every warp sums the 32 totals itself
  *sum = make_int2(__shfl_sync(0xffffffffu, w.x, 31), __shfl_sync(0xffffffffu, w.y, 31));
  const int bx = __shfl_sync(0xffffffffu, w.x, max(warp - 1, 0)), by = __shfl_sync(0xffffffffu, w.y, max(warp - 1, 0));
  return make_int2(x.x - v.x + (warp > 0 ? bx : 0), x.y - v.y + (warp > 0 ? by : 0));
}

__device__ __forceinline__ int pages_of(int tokens, int block_size) {
  return (int)(((long long)tokens + block_size - 1) / block_size);
}

__device__ void row_step(const PageParams& p) {
  static_assert(kPgThreads == 1024, "one warp total per lane in block_exclusive");
  __shared__ int2 warp_sums[32];
  __shared__ int had[kPgThreads];    // pages of a reset row (0: the row keeps its pages)
  __shared__ int count[kPgThreads];  // valid ones of them, then where they go on the stack
  __shared__ int list[kPgThreads];   // the reset rows that have pages, in any order: one warp each
  __shared__ int listed;
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
    if (threadIdx.x == 0) listed = 0;
    had[threadIdx.x] = old;
    count[threadIdx.x] = 0;
    __syncthreads();
    if (old > 0) list[atomicAdd(&listed, 1)] = threadIdx.x;
    __syncthreads();
    // a warp per reset row: how many of its entries name a page
    for (int i = warp; i < listed; i += kPgThreads / 32) {
      const int r = list[i];
      int n = 0;
      const int32_t* const row = p.table_in + (size_t)(b0 + r) * p.max_blocks;
#pragma unroll 8
      for (int j = lane; j < had[r]; j += 32) n += row[j] >= 0 && row[j] < p.num_blocks;
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) n += __shfl_xor_sync(0xffffffffu, n, d);
      if (lane == 0) count[r] = n;
    }
    __syncthreads();
    int2 sum;
    const int2 at = block_exclusive(make_int2(count[threadIdx.x], need), warp_sums, &sum);
    if (b < p.batch) {
      p.rows[b] = make_int4(start, fresh, kept, taken + at.y);
      p.seq_lens[b] = start + fresh;
    }
    count[threadIdx.x] = at.x;
    __syncthreads();
    for (int i = warp; i < listed; i += kPgThreads / 32) {
      const int r = list[i];
      long long to = (long long)free0 + pushed + count[r];
      const int32_t* const row = p.table_in + (size_t)(b0 + r) * p.max_blocks;
      for (int j0 = 0; j0 < had[r]; j0 += 32 * kPgAhead) {
        int e[kPgAhead];
#pragma unroll
        for (int k = 0; k < kPgAhead; ++k) {
          const int j = j0 + 32 * k + lane;
          e[k] = j < had[r] ? row[j] : -1;
        }
#pragma unroll
        for (int k = 0; k < kPgAhead; ++k) {
          const bool valid = e[k] >= 0 && e[k] < p.num_blocks;
          const uint32_t m = __ballot_sync(0xffffffffu, valid);
          const long long pos = to + __popc(m & ((1u << lane) - 1u));
          if (valid && pos < p.num_blocks) p.free_out[pos] = e[k];
          to += __popc(m);
        }
      }
    }
    pushed += sum.x;
    taken += sum.y;
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

// Four places of each list per thread and round: their loads are under way
// together (a round's latency is what a plan costs).
__device__ void fill_step(const PageParams& p, uint32_t first, uint32_t stride) {
  const int total = p.total[0], free0 = p.total[1];
  const bool in_place = p.table_out == p.table_in;
  // every count is below 2^31 and 4 strides at most 2^21: no index passes 2^32
  const uint32_t entries = (uint32_t)p.batch * (uint32_t)p.max_blocks;
  for (uint32_t i0 = first; i0 < entries; i0 += 4 * stride) {
    int b[4], j[4], v[4];
    int4 r[4];
    bool write[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t i = i0 + k * stride;
      write[k] = i < entries;
      b[k] = (int)(i / (uint32_t)p.max_blocks);
      j[k] = (int)(i - (uint32_t)b[k] * (uint32_t)p.max_blocks);
      if (write[k]) r[k] = p.rows[b[k]];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (!write[k]) continue;
      if (j[k] >= r[k].z && j[k] < pages_of(r[k].x + r[k].y, p.block_size))
        v[k] = taken_page(p, r[k].w + j[k] - r[k].z, total, free0);
      else if (p.reset != nullptr && p.reset[b[k]] != 0) v[k] = -1;
      else if (!in_place) v[k] = p.table_in[i0 + k * stride];
      else write[k] = false;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (write[k]) p.table_out[i0 + k * stride] = v[k];
  }
  const uint32_t tokens = (uint32_t)p.batch * (uint32_t)p.queries;
  for (uint32_t i0 = first; i0 < tokens; i0 += 4 * stride) {
    int pos[4], slot[4];
    int4 r[4];
    uint32_t b[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t i = i0 + k * stride;
      b[k] = i / (uint32_t)p.queries;
      pos[k] = (int)(i - b[k] * (uint32_t)p.queries);
      r[k] = i < tokens ? p.rows[b[k]] : make_int4(0, 0, 0, 0);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      pos[k] = pos[k] < r[k].y ? r[k].x + pos[k] : -1;
      slot[k] = -1;
      if (pos[k] >= 0) {  // pages that the row keeps are not written by this step
        const int j = pos[k] / p.block_size;
        if (j < r[k].z) {
          slot[k] = p.table_in[(size_t)b[k] * p.max_blocks + j];
          // the page that the row's first new token goes on in was missing in an earlier plan
          if (slot[k] == -1 && pos[k] == r[k].x) atomicAdd(p.missing, 1);
        } else {
          slot[k] = taken_page(p, r[k].w + j - r[k].z, total, free0);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t i = i0 + k * stride;
      if (i >= tokens) break;
      p.positions[i] = pos[k];
      p.lengths[i] = pos[k] + 1;
      p.slots[i] = slot[k] >= 0 && slot[k] < p.num_blocks ? slot[k] * p.block_size + pos[k] % p.block_size : -1;
    }
  }
  if (p.free_out != p.free_in)
    for (uint32_t i0 = first; i0 < (uint32_t)p.num_blocks; i0 += 4 * stride) {
      int v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t i = i0 + k * stride;
        if (i < (uint32_t)p.num_blocks) v[k] = p.free_in[i];
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t i = i0 + k * stride;
        if (i < (uint32_t)p.num_blocks && ((int)i < free0 || (int)i >= total)) p.free_out[i] = v[k];
      }
    }
}

__global__ void __launch_bounds__(kPgThreads) plan_rows_kernel(const PageParams p) { row_step(p); }

__global__ void __launch_bounds__(256) plan_fill_kernel(const PageParams p) {
  grid_dependency_wait();
  fill_step(p, blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
}

}  // namespace

cudaError_t launch_plan_pages(const PageParams& p, cudaStream_t stream) {
  plan_rows_kernel<<<1, kPgThreads, 0, stream>>>(p);
  cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  const long long work = (long long)p.batch * (p.max_blocks > p.queries ? p.max_blocks : p.queries);
  const long long most = work > p.num_blocks ? work : p.num_blocks;
  long long blocks = (most + 1023) / 1024;  // four places a thread
  if (blocks > 148 * 8) blocks = 148 * 8;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;  // plan_fill_kernel waits itself
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)blocks, 1, 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, plan_fill_kernel, p);
}

}  // namespace dsa
