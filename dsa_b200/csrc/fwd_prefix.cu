// tcgen05 attention of every query row over one dense key range that all of
// them share (a common prompt), and the join with partials over each query's
// own selected keys.
//
// Every (query, head) pair is a row, whatever query it belongs to: 128 rows
// are one MMA tile, and the keys need no gather. A cluster of two CTAs owns
// one item (row tile, key split) and walks its keys in tiles of 64:
//
//   score CTA (rank 0)  S = Q . K^T    M=128 rows, N=64 keys, K=576, Q in TMEM
//                       P = bf16(exp(S / scale_div - m)), online softmax
//   value CTA (rank 1)  O += P . V     M=128, N=2x256, K=64 keys, O fills TMEM
//
// O takes all 512 TMEM columns of an SM and Q 288 of another, as in the pair
// family, whose split of the work and lazy rescale (the factor is applied only
// when a row's maximum grows by more than 2^8) this kernel keeps.
//
// Keys come by TMA (one 3-D map that turns a row of 512 into eight 64-wide
// blocks, 128-byte swizzle) in half tiles of 64 keys x 256 dims (32 KB), each
// released by the MMAs that read it: two tiles of two halves in either CTA, and
// a rope block per tile in the score CTA. A box costs its issuer some
// 300 cycles whatever its size, so 8 KB boxes cannot keep a tile's pace (nine
// of them 3,200 cycles), and 32 KB ones can; whole tiles would keep fewer
// bytes in flight.
//
// P rounds the weights to BF16 for the MMA; the row sum adds them before the
// rounding, in FP32 (as every other family here).
//
// Roles (12 warps): score CTA 0 TMA, 1 and 3 QK issuers of the even and the
// odd tiles, 2 P sender, 4-11 softmax (warps 4-7 the even, 8-11 the odd tiles;
// the running maximum goes from one to the other); value CTA 0 TMA, 1 and 3 PV
// issuers of the lower and the upper 256 columns, 4-11 rescale and epilogue.
// Every wait is bounded and reports through the status word. No multicast
// loads.
#include <cuda.h>

#include <atomic>

#include "prefix.cuh"
#include "umma_ptx.cuh"

namespace dsa {
namespace {

using namespace umma;

constexpr int kPxThreads = 384;
constexpr int kPxRows = 128;
constexpr uint32_t kBlk = 64u * 128u;        // 64 keys x 64 dims, SW128
constexpr uint32_t kHalf = 4u * kBlk;        // 64 keys x 256 value columns
constexpr int kKParts = 3;                   // score CTA: dims 0-255, 256-511 and rope of a tile
constexpr int kKSlots = 2 * kKParts;         // two tiles
constexpr uint32_t kKTile = 2u * kHalf + kBlk;
constexpr int kVSlots = 4;                   // value CTA: ring of V half tiles, two tiles
constexpr int kSBufs = 2;                    // S buffer g % 2: QK issuer g % 2 fills it, softmax group g % 2 reads it
constexpr int kPSlots = 4;                   // value CTA
constexpr int kLSlots = 4;                   // score CTA: P staging (even: slot g % 4 is softmax group g % 2's)
constexpr uint32_t kPBytes = 128u * 64u * 2u;
constexpr uint32_t kAlphaOff = kPBytes;
constexpr uint32_t kFlagOff = kPBytes + 512u;
constexpr uint32_t kMsgBytes = kPBytes + 512u + 16u;
constexpr uint32_t kSlotBytes = kPBytes + 1024u;
constexpr uint32_t kFinBytes = 128u * 8u;
constexpr int kSoftWarp0 = 4;
constexpr int kEpiWarps = 8;

enum Bar {
  kKFull0 = 0,
  kKFree0 = kKFull0 + kKSlots,
  kQFull = kKFree0 + kKSlots,
  kSFull0,
  kSFree0 = kSFull0 + kSBufs,
  kMReady0 = kSFree0 + kSBufs,      // 4: per lane quadrant, the running max of the latest tile is posted
  kXchg0 = kMReady0 + 4,            // 4: per lane quadrant, both softmax warps posted their totals
  kLFull0 = kXchg0 + 4,             // P staging slot written (4 warps)
  kPDone0 = kLFull0 + kLSlots,      // PV that read the P slot is done (commit to both CTAs)
  kVFull0 = kPDone0 + kPSlots,
  kVFree0 = kVFull0 + kVSlots,
  kPFull0 = kVFree0 + kVSlots,      // P message landed
  kReq = kPFull0 + kPSlots,         // a rescale request is posted
  kReqDone,
  kFin,                             // (l, f) landed
  kDrain0,                          // 2: abort path, an issuer's MMAs are done
  kBarCount = kDrain0 + 2
};
// Arrivals that complete a phase.
__device__ __forceinline__ uint32_t bar_count(int i) {
  if (i == kQFull || i == kReqDone) return 8;                                  // softmax warps; epilogue warps
  if (i >= kSFree0 && i < kSFree0 + kSBufs) return 4;                          // the group's warps
  if (i >= kLFull0 && i < kLFull0 + kLSlots) return 4;
  if (i >= kXchg0 && i < kXchg0 + 4) return 2;                                 // both groups' warps of the quadrant
  if (i >= kPDone0 && i < kPDone0 + kPSlots) return 2;                         // both halves of the columns
  return 1;
}
constexpr uint32_t kOffTmemSlot = kBarCount * 8u;
constexpr uint32_t kOffAbort = kOffTmemSlot + 8u;
constexpr uint32_t kOffReq = kOffAbort + 8u;
constexpr uint32_t kOffData = 1024u;
constexpr uint32_t kOffLocal = kOffData + 2u * kKTile;              // score CTA
constexpr uint32_t kOffM = kOffLocal + kLSlots * kSlotBytes;       // [2][4 quads][32] running maxima
constexpr uint32_t kOffX = kOffM + 2u * 4u * 32u * 4u;             // [4 quads][2 warps][3][32] totals
constexpr uint32_t kScoreBytes = kOffX + 4u * 2u * 3u * 32u * 4u;
constexpr uint32_t kOffSlot = kOffData + kVSlots * kHalf;          // value CTA
constexpr uint32_t kOffFin = kOffSlot + kPSlots * kSlotBytes;
constexpr uint32_t kValueBytes = kOffFin + kFinBytes;
constexpr uint32_t kSmemBytes = (kScoreBytes > kValueBytes ? kScoreBytes : kValueBytes) + 1024u;
// The MMA cuts each of a score's 36 accumulations to FP32 instead of rounding
// it: half a unit in the last place is lost on average, 2^-25 to 2^-24 of a sum
// that has grown half way, together 36 / 2 * 2^-24.8 = 6e-7 of the score (5.6e-7
// measured, always towards zero). Scaling by 1 + 5.6e-7 takes the mean error of
// softmax_max from -5.6e-7 to below 1e-7 relative and with it that of softmax_sum,
// which is relative to the maximum, from 1.8e-6 to 5e-7.
constexpr double kCutBias = 5.6e-7;
constexpr uint32_t kReqEnd = 0xffffffffu;
constexpr uint32_t kTmemCols = 512, kTmemQ = 0, kTmemS = 288, kTmemO = 0;

static_assert(kOffReq + 8u <= kOffData && kBarCount <= kPxThreads, "barrier block");
static_assert(kEpiWarps == 8, "bar_count");
static_assert(kOffLocal % 1024 == 0 && kOffSlot % 1024 == 0 && kSlotBytes % 1024 == 0, "swizzle atoms");
static_assert(kSmemBytes <= 232448, "shared memory budget");
static_assert(kTmemS + kSBufs * 64 <= kTmemCols, "score TMEM budget");

__device__ __forceinline__ float u2f(uint32_t v) { return __uint_as_float(v); }
__device__ __forceinline__ uint32_t f2u(float v) { return __float_as_uint(v); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, volatile int* abort,
                                          bool cluster_scope = false) {
  const bool ok = mbar_wait(bar, parity, abort, cluster_scope);
  return __all_sync(0xffffffffu, ok) != 0;
}
__device__ __forceinline__ void st_async_b32x2(uint32_t remote_addr, uint32_t remote_bar, uint32_t a, uint32_t b) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];" ::"r"(
                   remote_addr),
               "r"(a), "r"(b), "r"(remote_bar)
               : "memory");
}
__device__ __forceinline__ void mma_commit_mc(uint32_t bar, uint16_t cta_mask) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          bar),
      "h"(cta_mask)
      : "memory");
}
// Box of the map at (0, row, blk) -> shared memory of this CTA.
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int row, int blk, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst),
      "l"(map), "r"(0), "r"(row), "r"(blk), "r"(bar)
      : "memory");
}

struct Maps {
  CUtensorMap half;  // latent, boxes of 64 keys x 256 dims
  CUtensorMap rope;  // rope, boxes of 64 keys x 64 dims
};

// Chunks [c0, c0 + N) (dims 64c..; chunk 8: rope) of the 32 Q rows of this
// warp -> TMEM, lane = row, 32 columns a chunk. The loads take whole 128-byte
// lines, four rows an instruction (a lane reading its own row costs 32 line
// lookups an instruction: 8,900 cycles for Q against 2,500), all chunks in flight
// together; each goes through 4 KB of shared memory (swizzled) to become rows.
template <int N>
__device__ __forceinline__ void load_q_chunks(const PrefixParams& p, long long row0, int lane, int c0, uint4 (*v)[8]) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const size_t row = (size_t)min(row0 + 4 * k + (lane >> 3), p.rows - 1);  // rows past the end repeat the last one
      v[i][k] = __ldg((c0 + i < 8 ? reinterpret_cast<const uint4*>(p.q + row * kDimLatent) + (c0 + i) * 8
                                  : reinterpret_cast<const uint4*>(p.q_rope + row * kDimRope)) + (lane & 7));
    }
}
template <int N>
__device__ __forceinline__ void store_q_chunks(int lane, int c0, const uint4 (*v)[8], uint8_t* scratch, uint32_t tq) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int r = 4 * k + (lane >> 3);
      *reinterpret_cast<uint4*>(scratch + r * 128 + (((lane & 7) ^ (r & 7)) * 16)) = v[i][k];
    }
    __syncwarp();
    uint32_t out[32];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint4 w = *reinterpret_cast<const uint4*>(scratch + lane * 128 + ((k ^ (lane & 7)) * 16));
      out[4 * k] = w.x;
      out[4 * k + 1] = w.y;
      out[4 * k + 2] = w.z;
      out[4 * k + 3] = w.w;
    }
    tmem_st32(tq + (uint32_t)(c0 + i) * 32u, out);
    __syncwarp();
  }
}

// Split cluster barrier: what this thread wrote before the arrive is visible
// to the peer's threads after their wait.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }

__global__ void __launch_bounds__(kPxThreads, 1) fwd_prefix_kernel(const PrefixParams p,
                                                                   const __grid_constant__ Maps maps) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* const sbase = smem_raw + (base - raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int item = (int)(blockIdx.x >> 1);
  const int mt = item / p.split, sp = item - mt * p.split;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sbase + kOffAbort);
  auto bar = [&](int i) -> uint32_t { return base + 8u * (uint32_t)i; };
  grid_launch_dependents();  // the own keys' kernel needs nothing from this one

  // keys [tile0 * 64, ...) of the split: whole tiles of the keys in use
  const int used = p.length != nullptr ? min(max(__ldg(p.length), 0), p.keys) : p.keys;
  const int all_tiles = (used + 63) / 64;
  const int tile0 = (int)((long long)all_tiles * sp / p.split);
  const int ntiles = (int)((long long)all_tiles * (sp + 1) / p.split) - tile0;
  const bool direct = p.part_num == nullptr;
  const long long row0 = (long long)mt * kPxRows;

  if (ntiles == 0) {  // the same in both CTAs: nothing to attend to
    for (int r = threadIdx.x; r < kPxRows; r += kPxThreads) {
      if (rank == 0 && direct && row0 + r < p.rows) {
        p.out_max[row0 + r] = -INFINITY;
        p.out_sum[row0 + r] = 0.f;
      } else if (rank == 0 && !direct) {
        p.part_max[(size_t)item * kPxRows + r] = kNegFltMax;
        p.part_sum[(size_t)item * kPxRows + r] = 0.f;  // the join does not read the numerator then
      }
    }
    if (rank == 1 && direct)
      for (int c = threadIdx.x; c < kPxRows * 64; c += kPxThreads)
        if (row0 + (c >> 6) < p.rows)
          reinterpret_cast<uint4*>(p.out + (row0 + (c >> 6)) * kDimLatent)[c & 63] = make_uint4(0, 0, 0, 0);
    return;
  }

  // the softmax warps' first two chunks of Q are under way while the CTA sets up
  uint4 q_first[3][8];
  if (rank == 0 && warp >= kSoftWarp0)
    load_q_chunks<2>(p, row0 + (warp & 3) * 32, lane, 5 * ((warp - kSoftWarp0) >> 2), q_first);
  // one barrier per thread (each CTA uses its own part of them)
  if (threadIdx.x < kBarCount) mbar_init(bar((int)threadIdx.x), bar_count((int)threadIdx.x));
  if (threadIdx.x == 0) *abort_flag = 0;
  fence_barrier_init();
  if (warp == 0) {
    tmem_alloc(base + kOffTmemSlot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(sbase + kOffTmemSlot);
  if (rank == 1 && threadIdx.x == 0) {
    for (int s = 0; s < kPSlots; ++s) mbar_arrive_expect_tx(bar(kPFull0 + s), kMsgBytes);
    mbar_arrive_expect_tx(bar(kFin), kFinBytes);
  }
  __syncwarp();
  // Each role waits for the peer CTA's barriers before it first addresses the
  // peer, or at its end; loads and Q start without it.
  cluster_arrive();

  bool ok = true;
  if (rank == 0) {
    // =============================== score CTA ===============================
    if (warp == 0) {
      // ---- TMA: part j of tile t into slot 3 (t % 2) + j; one thread ----
      if (lane == 0) {
        int t = 0, j = 0;
        for (; t < ntiles; ++t) {
          const uint32_t s0 = (uint32_t)(t & 1) * kKParts, stage = base + kOffData + (uint32_t)(t & 1) * kKTile;
          for (j = 0; j < kKParts; ++j) {
            if (t >= 2 && !(ok = mbar_wait(bar(kKFree0 + s0 + j), (uint32_t)((t >> 1) - 1) & 1u, abort_flag))) break;
            mbar_arrive_expect_tx(bar(kKFull0 + s0 + j), j < 2 ? kHalf : kBlk);
            tma_load_3d(stage + (uint32_t)j * kHalf, j < 2 ? &maps.half : &maps.rope, (tile0 + t) * 64, j < 2 ? 4 * j : 0,
                        bar(kKFull0 + s0 + j));
          }
          if (!ok) break;
        }
        if (!ok)  // loads in flight land before the CTA's memory goes
          for (int n = max(0, kKParts * t + j - kKSlots); n < kKParts * t + j; ++n)
            mbar_wait_drain(bar(kKFull0 + n % kKSlots), (uint32_t)(n / kKSlots) & 1u);
      }
      __syncwarp();
      cluster_wait();
    } else if (warp == 1 || warp == 3) {
      // ---- QK issuer i: S buffer i <- Q . K^T for tiles g = i mod 2, part by part (an issuer is held while
      // its MMAs run; the other one's waits fall into that time) ----
      const int i = warp >> 1;
      const uint32_t idesc = idesc_bf16(128, 64, false, false);
      ok = wait_warp(bar(kQFull), 0u, abort_flag);
      tc_fence_after();
      const uint32_t d = tmem + kTmemS + (uint32_t)i * 64u;
      const uint32_t s0 = (uint32_t)(i * kKParts);
      const uint64_t bd = smem_desc(base + kOffData + (uint32_t)i * kKTile, 16, 1024, kLayoutSw128);
      for (int g = i; g < ntiles && ok; g += 2) {
        if (g >= 2 && !(ok = wait_warp(bar(kSFree0 + i), (uint32_t)((g >> 1) - 1) & 1u, abort_flag))) break;
#pragma unroll
        for (int part = 0; part < kKParts; ++part) {
          if (!(ok = wait_warp(bar(kKFull0 + s0 + part), (uint32_t)(g >> 1) & 1u, abort_flag))) break;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int j = 4 * part; j < (part < 2 ? 4 * part + 4 : 9); ++j)
#pragma unroll
              for (int k = 0; k < 4; ++k)  // offsets in the descriptor's 16-byte units; 16 dims are 32 bytes
                mma_bf16_ts(d, tmem + kTmemQ + (uint32_t)(j * 4 + k) * 8u, bd + (uint64_t)(j * (kBlk / 16u) + 2 * k), idesc,
                            (j | k) ? 1u : 0u);
            mma_commit(bar(kKFree0 + s0 + part));
            if (part == kKParts - 1) mma_commit(bar(kSFull0 + i));
          }
          __syncwarp();
        }
      }
      if (!ok) {
        if (elect_one()) mma_commit(bar(kDrain0 + i));
        __syncwarp();
        mbar_wait_drain(bar(kDrain0 + i), 0u);
      }
      __syncwarp();
      cluster_wait();
    } else if (warp == 2) {
      // ---- P sender: staging slot g % 4 -> the value CTA's P slot g % 4 ----
      const uint32_t r_slot0 = mapa_shared(base + kOffSlot, 1);
      const uint32_t r_pfull0 = mapa_shared(bar(kPFull0), 1);
      cluster_wait();
      int g = 0;
      for (; g < ntiles; ++g) {
        const uint32_t ls = (uint32_t)g % kLSlots, ps = (uint32_t)g % kPSlots;
        if (!(ok = wait_warp(bar(kLFull0 + ls), (uint32_t)(g / kLSlots) & 1u, abort_flag))) break;
        if (g >= kPSlots && !(ok = wait_warp(bar(kPDone0 + ps), (uint32_t)(g / kPSlots - 1) & 1u, abort_flag))) break;
        if (lane == 0)
          bulk_copy_to_peer(r_slot0 + ps * kSlotBytes, base + kOffLocal + ls * kSlotBytes, kMsgBytes,
                            r_pfull0 + 8u * ps);
        __syncwarp();
      }
      // the value CTA's last commits arrive in this CTA's memory
      for (int k = max(0, ntiles - kPSlots); k < ntiles && ok; ++k)
        ok = wait_warp(bar(kPDone0 + k % kPSlots), (uint32_t)(k / kPSlots) & 1u, abort_flag);
    } else if (warp >= kSoftWarp0) {
      // ---- softmax: one row per thread; group e takes tiles g % 2 == e ----
      const int quad = warp & 3;
      const int e = (warp - kSoftWarp0) >> 2;
      const int row = quad * 32 + lane;
      const uint32_t t_lane = (uint32_t)(quad * 32) << 16;
      const float c = p.scale_log2;
      float* const mpub = reinterpret_cast<float*>(sbase + kOffM);
      float* const xch = reinterpret_cast<float*>(sbase + kOffX);
      {
        // scratch in the P staging slots: P of a tile is written after every warp's Q is loaded
        uint8_t* const scratch = sbase + kOffLocal + (warp - kSoftWarp0) * 4096;
        const uint32_t tq = tmem + t_lane + kTmemQ;
        store_q_chunks<2>(lane, 5 * e, q_first, scratch, tq);
        if (e == 0) {
          load_q_chunks<3>(p, row0 + quad * 32, lane, 2, q_first);
          store_q_chunks<3>(lane, 2, q_first, scratch, tq);
        } else {
          load_q_chunks<2>(p, row0 + quad * 32, lane, 7, q_first);
          store_q_chunks<2>(lane, 7, q_first, scratch, tq);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kQFull));
        cluster_wait();
      }
      float m_w = kNegFltMax, m_true = kNegFltMax, l = 0.f;
      for (int g = e; g < ntiles; g += 2) {
        const uint32_t b = (uint32_t)g % kSBufs;
        if (!(ok = wait_warp(bar(kSFull0 + b), (uint32_t)(g / kSBufs) & 1u, abort_flag))) break;
        tc_fence_after();
        float x[64];
        {
          uint32_t sv[64];
          tmem_ld32(tmem + t_lane + kTmemS + b * 64u, sv);
          tmem_ld32(tmem + t_lane + kTmemS + b * 64u + 32u, sv + 32);
          tmem_wait_ld_regs32(sv);
          tmem_wait_ld_regs32(sv + 32);
#pragma unroll
          for (int k = 0; k < 64; ++k) x[k] = u2f(sv[k]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kSFree0 + b));
        const int valid = used - (tile0 + g) * 64;
        if (valid < 64) {
#pragma unroll
          for (int k = 0; k < 64; ++k) x[k] = k < valid ? x[k] : -INFINITY;
        }
        float mx;
        {
          float r[32];
#pragma unroll
          for (int k = 0; k < 32; ++k) r[k] = fmaxf(x[k], x[k + 32]);
#pragma unroll
          for (int w = 16; w >= 1; w >>= 1)
#pragma unroll
            for (int k = 0; k < w; ++k) r[k] = fmaxf(r[k], r[k + w]);
          mx = r[0];
        }
        m_true = fmaxf(m_true, mx);
        float m_prev = kNegFltMax;
        if (g > 0) {
          if (!(ok = wait_warp(bar(kMReady0 + quad), (uint32_t)(g - 1) & 1u, abort_flag))) break;
          m_prev = mpub[(((g - 1) & 1) * 4 + quad) * 32 + lane];
        }
        const float m_t = ((mx - m_prev) * c > 8.f) ? mx : m_prev;  // lazy rescale threshold 2^8
        mpub[((g & 1) * 4 + quad) * 32 + lane] = m_t;
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kMReady0 + quad));
        const bool resc = g > 0 && m_t != m_prev;  // the first PV overwrites O
        const float alpha = resc ? ex2((m_prev - m_t) * c) : 1.f;
        const float mc = m_t * c;
        uint32_t packed[32];
        float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll
        for (int k = 0; k < 64; k += 4) {
          const float p0 = ex2(fmaf(x[k], c, -mc)), p1 = ex2(fmaf(x[k + 1], c, -mc));
          const float p2 = ex2(fmaf(x[k + 2], c, -mc)), p3 = ex2(fmaf(x[k + 3], c, -mc));
          s0 += p0;
          s1 += p1;
          s2 += p2;
          s3 += p3;
          packed[k / 2] = pack_bf16x2(p0, p1);
          packed[k / 2 + 1] = pack_bf16x2(p2, p3);
        }
        if (m_t != m_w) {
          l *= ex2((m_w - m_t) * c);
          m_w = m_t;
        }
        l += (s0 + s1) + (s2 + s3);
        const uint32_t flag = __any_sync(0xffffffffu, resc) ? 1u : 0u;
        // the staging slot's message of tile g - 4 has landed: its PV is done
        if (g >= kLSlots) {
          const uint32_t gp = (uint32_t)(g - kLSlots);
          if (!(ok = wait_warp(bar(kPDone0 + gp % kPSlots), (gp / kPSlots) & 1u, abort_flag))) break;
        }
        const uint32_t ls = (uint32_t)g % kLSlots;
        uint8_t* const slot = sbase + kOffLocal + ls * kSlotBytes;
        uint8_t* const prow = slot + (uint32_t)(row >> 3) * 1024u + (uint32_t)(row & 7) * 128u;
#pragma unroll
        for (int q = 0; q < 8; ++q)
          *reinterpret_cast<uint4*>(prow + (uint32_t)((q ^ (row & 7)) * 16)) =
              make_uint4(packed[4 * q], packed[4 * q + 1], packed[4 * q + 2], packed[4 * q + 3]);
        *reinterpret_cast<float*>(slot + kAlphaOff + (uint32_t)row * 4u) = alpha;
        if (lane == 0) *reinterpret_cast<uint32_t*>(slot + kFlagOff + (uint32_t)quad * 4u) = flag;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kLFull0 + ls));
      }
      // ---- totals of the two groups ----
      if (ok) {
        float* const mine = xch + (quad * 2 + e) * 96;
        const float* const other = xch + (quad * 2 + (e ^ 1)) * 96;
        mine[lane] = m_w;
        mine[32 + lane] = l;
        mine[64 + lane] = m_true;
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kXchg0 + quad));
        ok = wait_warp(bar(kXchg0 + quad), 0u, abort_flag);
        if (ok && e == 0) {
          const float m_o = other[lane], l_o = other[32 + lane];
          const float m_fin = fmaxf(m_w, m_o);
          l = (m_w == m_fin ? l : l * ex2((m_w - m_fin) * c)) + (m_o == m_fin ? l_o : l_o * ex2((m_o - m_fin) * c));
          m_true = fmaxf(m_true, other[64 + lane]);
          const float f = m_true == kNegFltMax ? 1.f : ex2((m_fin - m_true) * c);
          if (!direct) {
            const size_t pr = (size_t)item * kPxRows + row;
            p.part_max[pr] = m_true == kNegFltMax ? kNegFltMax : __fdiv_rn(m_true, p.scale_div);
            p.part_sum[pr] = l * f;
          } else if (row0 + row < p.rows) {
            p.out_max[row0 + row] = final_max(m_true, l, p.scale_div);
            p.out_sum[row0 + row] = l * f;
          }
          st_async_b32x2(mapa_shared(base + kOffFin, 1) + (uint32_t)row * 8u, mapa_shared(bar(kFin), 1), f2u(l), f2u(f));
        }
      }
    }
  } else {
    // =============================== value CTA ===============================
    if (warp == 0) {
      // ---- TMA: half tile n = 2 t + h into slot n % kVSlots; one thread ----
      if (lane == 0) {
        int n = 0;
        for (; n < 2 * ntiles; ++n) {
          const uint32_t s = (uint32_t)n % kVSlots;
          if (n >= kVSlots && !(ok = mbar_wait(bar(kVFree0 + s), (uint32_t)(n / kVSlots - 1) & 1u, abort_flag))) break;
          mbar_arrive_expect_tx(bar(kVFull0 + s), kHalf);
          tma_load_3d(base + kOffData + s * kHalf, &maps.half, (tile0 + (n >> 1)) * 64, (n & 1) * 4, bar(kVFull0 + s));
        }
        if (!ok)
          for (int k = max(0, n - kVSlots); k < n; ++k)
            mbar_wait_drain(bar(kVFull0 + k % kVSlots), (uint32_t)(k / kVSlots) & 1u);
      }
      __syncwarp();
      cluster_wait();
    } else if (warp == 1 || warp == 3) {
      // ---- PV issuer h: O[:, 256 h .. 256 h + 255] += P . V; issuer 0 posts the requests ----
      const int h = warp >> 1;
      cluster_wait();
      const uint32_t idesc = idesc_bf16(128, 256, false, true);
      volatile uint32_t* const req = reinterpret_cast<volatile uint32_t*>(sbase + kOffReq);
      uint32_t nresc = 0;
      for (int g = 0; g < ntiles && ok; ++g) {
        const uint32_t s = (uint32_t)g % kPSlots;
        if (!(ok = wait_warp(bar(kPFull0 + s), (uint32_t)(g / kPSlots) & 1u, abort_flag, true))) break;
        const uint32_t slot = base + kOffSlot + s * kSlotBytes;
        if (h == 0 && lane == 0 && g + kPSlots < ntiles) mbar_arrive_expect_tx(bar(kPFull0 + s), kMsgBytes);  // its next message
        __syncwarp();
        const volatile uint32_t* fl = reinterpret_cast<const volatile uint32_t*>(sbase + (slot - base) + kFlagOff);
        if ((fl[0] | fl[1] | fl[2] | fl[3]) != 0u) {
          if (h == 0 && lane == 0) {
            *req = (uint32_t)g;
            mbar_arrive(bar(kReq));
          }
          __syncwarp();
          if (!(ok = wait_warp(bar(kReqDone), nresc & 1u, abort_flag))) break;
          ++nresc;
        }
        const int valid = used - (tile0 + g) * 64;
        const uint32_t vs = (uint32_t)(2 * g + h) % kVSlots;
        if (!(ok = wait_warp(bar(kVFull0 + vs), (uint32_t)(g >> 1) & 1u, abort_flag))) break;
        const uint32_t vslot = base + kOffData + vs * kHalf;
        if (valid < 64) {
          // rows behind the last key: weight 0, but 0 x NaN of a cache row never written would not be 0
          for (int i = lane; i < (64 - valid) * 32; i += 32) {
            const int r = valid + (i >> 5), q = i & 31;
            *reinterpret_cast<uint4*>(sbase + (vslot - base) + (uint32_t)(q >> 3) * kBlk + (uint32_t)r * 128u +
                                      (uint32_t)(q & 7) * 16u) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            mma_bf16_ss(tmem + kTmemO + h * 256, smem_desc(slot + j * 32, 16, 1024, kLayoutSw128),
                        smem_desc(vslot + j * 2048, kBlk, 1024, kLayoutSw128), idesc, (g | j) ? 1u : 0u);
          mma_commit(bar(kVFree0 + vs));
          mma_commit_mc(bar(kPDone0 + s), (uint16_t)3);
        }
        __syncwarp();
      }
      if (ok) {
        if (h == 0 && lane == 0) {
          *req = kReqEnd;
          mbar_arrive(bar(kReq));
        }
        __syncwarp();
      } else {
        if (elect_one()) mma_commit(bar(kDrain0 + h));
        __syncwarp();
        mbar_wait_drain(bar(kDrain0 + h), 0u);
      }
    } else if (warp >= kSoftWarp0) {
      // ---- rescale requests, then the epilogue: half `part` of the columns of 32 rows ----
      const int quad = warp & 3, part = (warp - kSoftWarp0) >> 2;
      cluster_wait();
      const int row = quad * 32 + lane;
      const uint32_t t_o = tmem + ((uint32_t)(quad * 32) << 16) + kTmemO + (uint32_t)part * 256u;
      const volatile uint32_t* const req = reinterpret_cast<const volatile uint32_t*>(sbase + kOffReq);
      auto pv_done = [&](int g) { return wait_warp(bar(kPDone0 + g % kPSlots), (uint32_t)(g / kPSlots) & 1u, abort_flag); };
      for (uint32_t nreq = 0;; ++nreq) {
        if (!(ok = wait_warp(bar(kReq), nreq & 1u, abort_flag))) break;
        const uint32_t g = *req;
        if (g == kReqEnd) break;
        const uint8_t* slot = sbase + kOffSlot + (g % kPSlots) * kSlotBytes;
        const uint32_t flag = *reinterpret_cast<const volatile uint32_t*>(slot + kFlagOff + quad * 4);
        if (flag != 0u) {
          const float alpha = *reinterpret_cast<const volatile float*>(slot + kAlphaOff + row * 4);
          if (!(ok = pv_done((int)g - 1))) break;
          tc_fence_after();
#pragma unroll 1
          for (int cb = 0; cb < 256; cb += 32) {
            uint32_t o[32];
            tmem_ld32(t_o + (uint32_t)cb, o);
            tmem_wait_ld_regs32(o);
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = f2u(u2f(o[k]) * alpha);
            tmem_st32(t_o + (uint32_t)cb, o);
          }
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kReqDone));
      }
      if (ok && (ok = wait_warp(bar(kFin), 0u, abort_flag, true)) && (ok = pv_done(ntiles - 1))) {
        const volatile float* lf = reinterpret_cast<const volatile float*>(sbase + kOffFin + row * 8);
        const float l = lf[0], f = lf[1];
        tc_fence_after();
        const long long grow = row0 + row;
        if (direct) {
          const float rl = l > 0.f || l != l ? __frcp_rn(l) : 0.f;
          __nv_bfloat16* const dst = p.out + (size_t)(grow & ~1LL) * kDimLatent + part * 256;
          const bool wide = (reinterpret_cast<uintptr_t>(p.out) & 31u) == 0;
#pragma unroll 1
          for (int cb = 0; cb < 256; cb += 32) {
            uint32_t o[32];
            tmem_ld32(t_o + (uint32_t)cb, o);
            tmem_wait_ld_regs32(o);
            uint32_t a[8], b[8];
            pack_bf16_row32_paired(o, rl, a, b);
            if (grow < p.rows) store_bf16_row32_paired(dst + cb, kDimLatent, a, b, wide);  // rows is even: pairs are whole
          }
        } else {
          // [64 groups of 8 columns][128 rows][8]: a store instruction writes 1 KB in a row
          float* const dst = p.part_num + ((size_t)item * 64 + part * 32) * (kPxRows * 8) + row * 8;
          const bool live = grow < p.rows;
#pragma unroll 1
          for (int cb = 0; cb < 256 && row0 + quad * 32 < p.rows; cb += 64) {
            uint32_t o[64];
            tmem_ld32(t_o + (uint32_t)cb, o);
            tmem_ld32(t_o + (uint32_t)cb + 32u, o + 32);
            tmem_wait_ld_regs32(o);
            tmem_wait_ld_regs32(o + 32);
#pragma unroll
            for (int k = 0; k < 64; ++k) o[k] = f2u(u2f(o[k]) * f);
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (live) st_global_v8(dst + (size_t)(cb / 8 + k) * (kPxRows * 8), o + 8 * k);
          }
        }
        tc_fence_before();
      }
    } else {
      cluster_wait();
    }
  }
  if (!ok && lane == 0) report_error(p.status, kErrTimeout);
  __syncwarp();
  tc_fence_before();
  cluster_sync();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Join of a row's prefix partials and its own-key partials: m = max m_i,
// out = sum_i e^(m_i - m) n_i / sum_i e^(m_i - m) l_i. A block takes 32 rows
// (lane = row) and 64 columns (8 a warp) and shares its rows' (m, l) in shared
// memory. Bound by the partials' 2 KB a row and part, and with few rows by
// latency: a thread's first four parts are under way before the weights are
// known (8192 rows of 3 parts 20 -> 15 us from DRAM; eight in flight cost
// occupancy, 21 us). A part of weight 0 counts as 0 whatever its numerator
// holds (nothing is written there when it has no keys).
constexpr int kJoinWarps = 8;
constexpr int kJoinMaxParts = 160;

__global__ void __launch_bounds__(32 * kJoinWarps) prefix_join_kernel(const JoinParams p) {
  __shared__ float2 stats[kJoinMaxParts][32];
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long r = (long long)blockIdx.x * 32 + lane;
  const bool live = r < p.rows;
  const long long rr = live ? r : p.rows - 1;
  const int n = p.split + p.own_split;
  const long long token = rr / p.heads;
  const long long px0 = (rr >> 7) * p.split;                                 // + part: [.., 128] rows
  const long long own0 = token * p.own_split * p.heads + (rr - token * p.heads);  // + part * heads
  const int col = blockIdx.y * (8 * kJoinWarps) + warp * 8;
  const float* const px_src = p.part_num + ((size_t)px0 * 64 + col / 8) * (kPxRows * 8) + (rr & 127) * 8;
  const float* const own_src = p.own_num + (size_t)own0 * kDimLatent + col;
  float4 v[4][2];
  auto load4 = [&](int i0) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + j;
      if (i < n) {
        const float* const src = i < p.split ? px_src + (size_t)i * (64 * kPxRows * 8)
                                             : own_src + (size_t)(i - p.split) * p.heads * kDimLatent;
        v[j][0] = reinterpret_cast<const float4*>(src)[0];
        v[j][1] = reinterpret_cast<const float4*>(src)[1];
      }
    }
  };
  load4(0);
  for (int i = warp; i < n; i += kJoinWarps) {
    const bool px = i < p.split;
    const long long k = px ? (px0 + i) * kPxRows + (rr & 127) : own0 + (long long)(i - p.split) * p.heads;
    stats[i][lane] = px ? make_float2(p.part_max[k], p.part_sum[k]) : make_float2(p.own_max[k], p.own_sum[k]);
  }
  __syncthreads();
  float top = kNegFltMax;
  for (int i = 0; i < n; ++i) {
    const float2 ml = stats[i][lane];
    if (ml.y != 0.f) top = fmaxf(top, ml.x);
  }
  float acc[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) acc[k] = 0.f;
  float total = 0.f;
  for (int i0 = 0; i0 < n; i0 += 4) {
    if (i0 > 0) load4(i0);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 ml = i0 + j < n ? stats[i0 + j][lane] : make_float2(0.f, 0.f);
      const float w = ml.y != 0.f ? expf(ml.x - top) : 0.f;
      if (w != 0.f) {
        total = fmaf(w, ml.y, total);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          acc[4 * h] = fmaf(w, v[j][h].x, acc[4 * h]);
          acc[4 * h + 1] = fmaf(w, v[j][h].y, acc[4 * h + 1]);
          acc[4 * h + 2] = fmaf(w, v[j][h].z, acc[4 * h + 2]);
          acc[4 * h + 3] = fmaf(w, v[j][h].w, acc[4 * h + 3]);
        }
      }
    }
  }
  if (!live) return;
  const float rl = total != 0.f ? __frcp_rn(total) : 0.f;
  *reinterpret_cast<uint4*>(p.out + r * kDimLatent + col) =
      make_uint4(pack_bf16x2(acc[0] * rl, acc[1] * rl), pack_bf16x2(acc[2] * rl, acc[3] * rl),
                 pack_bf16x2(acc[4] * rl, acc[5] * rl), pack_bf16x2(acc[6] * rl, acc[7] * rl));
  if (col == 0) {
    p.out_max[r] = total != 0.f ? top : -INFINITY;
    p.out_sum[r] = total;
  }
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeFn>(f);
  }();
  return fn;
}

// `rows` rows of blocks x 64 elements as [blocks][rows][64], boxes of
// box_blocks x 64 rows x 64.
bool encode(CUtensorMap* map, const void* ptr, long long rows, int blocks, int box_blocks) {
  const EncodeFn fn = encode_fn();
  if (fn == nullptr) return false;
  const cuuint64_t dims[3] = {64, (cuuint64_t)rows, (cuuint64_t)blocks};
  const cuuint64_t strides[2] = {(cuuint64_t)blocks * 128u, 128u};
  const cuuint32_t box[3] = {64, 64, (cuuint32_t)box_blocks};
  const cuuint32_t ones[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(ptr), dims, strides, box, ones,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool launch_config(cudaLaunchConfig_t* cfg, cudaLaunchAttribute* attr, unsigned ctas, cudaStream_t stream) {
  // once per device: the attribute belongs to the device's context
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if ((ready.load(std::memory_order_relaxed) & bit) == 0) {
    if (cudaFuncSetAttribute(fwd_prefix_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBytes) != cudaSuccess)
      return false;
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  attr->id = cudaLaunchAttributeClusterDimension;
  attr->val.clusterDim.x = 2;
  attr->val.clusterDim.y = 1;
  attr->val.clusterDim.z = 1;
  *cfg = cudaLaunchConfig_t{};
  cfg->gridDim = dim3(ctas, 1, 1);
  cfg->blockDim = dim3(kPxThreads, 1, 1);
  cfg->dynamicSmemBytes = kSmemBytes;
  cfg->stream = stream;
  cfg->attrs = attr;
  cfg->numAttrs = 1;
  return true;
}

}  // namespace

int prefix_max_clusters() {
  static int cached = -1;
  if (cached > 0) return cached;
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr;
  int n = 0;
  if (!launch_config(&cfg, &attr, 148, nullptr) ||
      cudaOccupancyMaxActiveClusters(&n, fwd_prefix_kernel, &cfg) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    return -1;
  }
  cached = n;
  return cached;
}

cudaError_t launch_fwd_prefix(const PrefixParams& p, const void* kv, const void* k_rope, cudaStream_t stream) {
  Maps maps;
  if (!encode(&maps.half, kv, p.keys, 8, 4) || !encode(&maps.rope, k_rope, p.keys, 1, 1))
    return cudaErrorInvalidValue;
  PrefixParams scaled = p;
  scaled.scale_div = (float)(p.scale_div * (1.0 - kCutBias));
  scaled.scale_log2 = (float)(p.scale_log2 * (1.0 + kCutBias));
  const long long items = (p.rows + kPxRows - 1) / kPxRows * p.split;
  if (items <= 0 || 2 * items > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr;
  if (!launch_config(&cfg, &attr, (unsigned)(2 * items), stream)) return cudaErrorInvalidConfiguration;
  return cudaLaunchKernelEx(&cfg, fwd_prefix_kernel, scaled, maps);
}

cudaError_t launch_prefix_join(const JoinParams& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;  // its start overlaps the end of the kernel before it
  attr.val.programmaticStreamSerializationAllowed = 1;
  if (p.split + p.own_split > kJoinMaxParts) return cudaErrorInvalidValue;
  cfg.gridDim = dim3((unsigned)((p.rows + 31) / 32), kDimLatent / (8 * kJoinWarps), 1);
  cfg.blockDim = dim3(32 * kJoinWarps, 1, 1);
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, prefix_join_kernel, p);
}

}  // namespace dsa
