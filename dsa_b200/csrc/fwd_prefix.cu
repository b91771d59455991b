// tcgen05 attention of every query row over one dense key range that all of
// them share (a common prompt), and the join with partials over each query's
// own selected keys.
//
// Every (query, head) pair is a row, whatever query it belongs to: 128 rows
// are one MMA tile, and the keys need no gather. A cluster of G score CTAs and
// G value CTAs (G = 1 or 2) owns one item (G row tiles, key split) and walks
// its keys in tiles of 64:
//
//   score CTAs (ranks 0 .. G-1)   S = Q . K^T   M=128 G rows, N=64 keys, K=576, Q in TMEM
//                                 P = bf16(exp(S / scale_div - m)), online softmax
//   value CTAs (ranks G .. 2G-1)  O += P . V    M=128 G, N=2x256, K=64 keys, O fills TMEM
//
// O takes all 512 TMEM columns of an SM and Q 288 of another, as in the pair
// family, whose split of the work and lazy rescale (the factor is applied only
// when a row's maximum grows by more than 2^8) this kernel keeps.
//
// With G = 2 the MMAs pair the SMs (cta_group::2): each SM holds half of the K
// or V tile and both tensor cores read the two halves, so a tile costs an SM
// half the shared memory traffic and half the L2 reads. That traffic is what
// bounds G = 1: a tile writes and reads 72 KB of K and passes 17 KB of P in the
// score CTA, writes and reads 64 KB of V and reads P twice in the value CTA,
// 178 KB each at 128 bytes a cycle = 1,390 cycles (1,400 measured) against
// 1,152 of MMA. G = 2 takes 1,190: 4096 rows over 32003 keys run at 1,480
// TFLOP/s (0.89 of the measured cuBLAS burst, 1.08 of its sustained rate; G = 1
// 1,170), 1024 rows over 32768, in eight splits, at 1,207 (G = 1 1,030).
//
// Keys come by TMA (one 3-D map that turns a row of 512 into eight 64-wide
// blocks, 128-byte swizzle) in boxes of 32 KB / G, each released by the MMAs
// that read it. A box costs its issuer some 300 cycles whatever its size, so
// 8 KB boxes could not keep a tile's pace.
//
// P rounds the weights to BF16 for the MMA; the row sum adds them before the
// rounding, in FP32 (as every other family here). A score is 36 accumulations
// of the MMA, each cut to FP32: it is exact where the sums of the products are,
// within 36 * 2^-23 of its partial sums' size anywhere, and on random data
// 5.6e-7 of itself too near to zero on average (softmax_sum then 1.8e-6 too
// large; an FP32 product of torch's is 2e-7 and 7e-7 off), as in the pair
// family. Nothing corrects for it: the loss depends on the data, and the own
// keys' scores, which share the softmax, lose theirs alike. Two sums a score
// (dims 0-255, the rest; three S buffers fit the TMEM) halve the loss, 7.7e-7
// on the sum, but the second buffer's reads and its turn-around take 13 % of
// 4096 rows over 32003 keys (201 -> 228 us) and 11 % of 1024 over 32768.
//
// Roles (12 warps; the MMAs of a pair are issued by its first CTA): score CTA
// 0 TMA, 1 and 3 QK issuers of the even and the odd tiles, in turn (an issuer
// is held while its MMAs run; the other one's waits fall into that time), 2 P sender,
// 4-11 softmax (warps 4-7 the even, 8-11 the odd tiles; the running maximum
// goes from one to the other); value CTA 0 TMA, 1 and 3 PV issuers of the lower
// and the upper 256 columns, 2 receives P (asks for a rescale where one is due,
// clears what lies behind the last key) and tells the issuers, 4-11 rescale and
// epilogue. Every wait is bounded and reports through the status word. No
// multicast loads.
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
constexpr int kKParts = 3;                   // dims 0-255, 256-511 and rope of a tile
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
constexpr uint32_t kReqEnd = 0xffffffffu;
constexpr uint32_t kTmemCols = 512, kTmemQ = 0, kTmemS = 288, kTmemO = 0;

// Sizes and barriers that depend on the CTAs of a pair. "Leader": the barrier
// of the pair's first CTA is used by both.
template <int G>
struct Cfg {
  static constexpr uint32_t kKBlk = kBlk / G;                  // 64 / G keys x 64 dims
  static constexpr uint32_t kKTile = 9u * kKBlk;
  static constexpr int kKStages = 2 * G;                       // tiles in the score CTA (even: a stage belongs to one issuer)
  static constexpr uint32_t kVBox = 4u / G * kBlk;             // 64 keys x 256 / G columns of one half
  static constexpr int kVSlots = 4 * G;                        // half tiles in the value CTA (even, as above)
  enum Bar {
    kKFull0 = 0,                              // leader: a part of a tile has landed in both CTAs
    kKFree0 = kKFull0 + kKStages * kKParts,   // its MMAs are done (commit to the pair)
    kQFull = kKFree0 + kKStages * kKParts,    // leader: Q of both CTAs is in TMEM
    kTurn0,                                   // 2: leader's QK issuer i may issue its next tile
    kSFull0 = kTurn0 + 2,                     // commit to the pair
    kSFree0 = kSFull0 + kSBufs,               // leader: both CTAs have read S
    kMReady0 = kSFree0 + kSBufs,              // 4: per lane quadrant, the running max of the latest tile is posted
    kXchg0 = kMReady0 + 4,                    // 4: per lane quadrant, both softmax warps posted their totals
    kLFull0 = kXchg0 + 4,                     // P staging slot written (4 warps)
    kPDone0 = kLFull0 + kLSlots,              // PVs that read the P slot are done (commits to all CTAs)
    kVFull0 = kPDone0 + kPSlots,              // leader
    kVFree0 = kVFull0 + kVSlots,              // commit to the pair
    kVLast0 = kVFree0 + kVSlots,              // 2: the last, partly filled tile's halves have landed in this CTA
    kPFull0 = kVLast0 + 2,                    // P message landed
    kPReady0 = kPFull0 + kPSlots,             // leader: both CTAs' P (and O) are ready for the tile's PV
    kReq = kPReady0 + kPSlots,                // a rescale request is posted
    kReqDone,
    kFin,                                     // (l, f) landed
    kDrain0,                                  // 2: abort path, an issuer's MMAs are done
    kBarCount = kDrain0 + 2
  };
  // Arrivals that complete a phase.
  static __device__ __forceinline__ uint32_t bar_count(int i) {
    if (i == kQFull) return 8 * G;                                               // softmax warps
    if (i == kReqDone) return kEpiWarps;
    if (i >= kSFree0 && i < kSFree0 + kSBufs) return 4 * G;                      // the group's warps
    if (i >= kLFull0 && i < kLFull0 + kLSlots) return 4;
    if (i >= kXchg0 && i < kXchg0 + 4) return 2;                                 // both groups' warps of the quadrant
    if (i >= kPDone0 && i < kPDone0 + kPSlots) return 2;                         // both halves of the columns
    if (i >= kPReady0 && i < kPReady0 + kPSlots) return G;                       // the receivers
    return 1;
  }
  static constexpr uint32_t kOffTmemSlot = kBarCount * 8u;
  static constexpr uint32_t kOffAbort = kOffTmemSlot + 8u;
  static constexpr uint32_t kOffReq = kOffAbort + 8u;
  static constexpr uint32_t kOffData = 1024u;
  static constexpr uint32_t kOffLocal = kOffData + kKStages * kKTile;          // score CTA
  static constexpr uint32_t kOffM = kOffLocal + kLSlots * kSlotBytes;          // [2][4 quads][32] running maxima
  static constexpr uint32_t kOffX = kOffM + 2u * 4u * 32u * 4u;                // [4 quads][2 warps][3][32] totals
  static constexpr uint32_t kScoreBytes = kOffX + 4u * 2u * 3u * 32u * 4u;
  static constexpr uint32_t kOffSlot = kOffData + kVSlots * kVBox;             // value CTA
  static constexpr uint32_t kOffFin = kOffSlot + kPSlots * kSlotBytes;
  static constexpr uint32_t kValueBytes = kOffFin + kFinBytes;
  static constexpr uint32_t kSmemBytes = (kScoreBytes > kValueBytes ? kScoreBytes : kValueBytes) + 1024u;
  static_assert(kOffReq + 8u <= kOffData && kBarCount <= kPxThreads, "barrier block");
  static_assert(kOffLocal % 1024 == 0 && kOffSlot % 1024 == 0 && kSlotBytes % 1024 == 0, "swizzle atoms");
  static_assert(kSmemBytes <= 232448, "shared memory budget");
  static_assert(kTmemS + kSBufs * 64 <= kTmemCols, "score TMEM budget");
};

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

// Arrive on another CTA's barrier. What it reports is in this SM's tensor and
// shared memory, which the leader's MMAs use in place: a release at CTA scope
// is enough (one at cluster scope waits 1,000 to 2,000 cycles for the thread's
// other memory operations).
__device__ __forceinline__ void mbar_arrive_at(uint32_t remote_bar) {
  asm volatile("mbarrier.arrive.release.cta.shared::cluster.b64 _, [%0];" ::"r"(remote_bar) : "memory");
}

// tcgen05 instructions of a pair of G CTAs (all of a kernel's have one cta_group).
template <int G>
__device__ __forceinline__ void commit_to(uint32_t bar, uint16_t cta_mask) {
  if constexpr (G == 1)
    asm volatile(
        "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            bar),
        "h"(cta_mask)
        : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            bar),
        "h"(cta_mask)
        : "memory");
}
template <int G>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  if constexpr (G == 1)
    mma_bf16_ts(d, a_tmem, b_desc, idesc, accumulate);
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
template <int G>
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  if constexpr (G == 1)
    mma_bf16_ss(d, a_desc, b_desc, idesc, accumulate);
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
template <int G>
__device__ __forceinline__ void tmem_take(uint32_t dst) {
  if constexpr (G == 1) {
    tmem_alloc(dst, kTmemCols);
    tmem_relinquish();
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int G>
__device__ __forceinline__ void tmem_give(uint32_t taddr) {
  if constexpr (G == 1)
    tmem_dealloc(taddr, kTmemCols);
  else
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(kTmemCols) : "memory");
}
// Box of the map at (0, row, blk) -> shared memory of this CTA; completes on a
// barrier of this CTA, or (kPair) on one of its pair's first CTA.
template <bool kPair>
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int row, int blk, uint32_t bar) {
  if constexpr (!kPair)
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            dst),
        "l"(map), "r"(0), "r"(row), "r"(blk), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(map), "r"(0), "r"(row), "r"(blk), "r"(bar)
        : "memory");
}

struct Maps {
  CUtensorMap k;     // latent, boxes of 64 / G keys x 256 dims
  CUtensorMap v;     // latent, boxes of 64 keys x 256 / G dims
  CUtensorMap rope;  // rope, boxes of 64 / G keys x 64 dims
};

// Q of a warp's 32 rows -> TMEM, lane = row, 32 columns per chunk of 64 dims
// (chunk 8: rope). The loads take whole 128-byte lines, four rows an
// instruction (a lane reading its own row costs 32 line lookups an instruction:
// 8,900 cycles for Q), and all of a warp's chunks are in flight together, two
// into shared memory and the rest into registers; a chunk goes through 4 KB of
// shared memory (swizzled) to become rows.
struct QRows {
  const uint8_t *latent, *rope;  // this lane's 16 bytes of the warp's first row
  int first, last;               // this lane's row of piece 0, the last row that is there (later ones repeat it)
  __device__ __forceinline__ QRows(const PrefixParams& p, long long row0, int lane) {
    const long long at = min(row0, p.rows - 1);
    latent = reinterpret_cast<const uint8_t*>(p.q + at * kDimLatent) + (lane & 7) * 16;
    rope = reinterpret_cast<const uint8_t*>(p.q_rope + at * kDimRope) + (lane & 7) * 16;
    first = lane >> 3;
    last = (int)min(p.rows - 1 - at, 31LL);
  }
  __device__ __forceinline__ const uint4* piece(int c, int k) const {  // rows 4 k ..  of chunk c
    const int r = min(first + 4 * k, last);
    return reinterpret_cast<const uint4*>(c < 8 ? latent + r * 1024 + c * 128 : rope + r * 128);
  }
};
__device__ __forceinline__ uint32_t q_place(int lane, int k) {  // of piece k of a chunk in its 4 KB
  const int r = 4 * k + (lane >> 3);
  return (uint32_t)(r * 128 + (((lane & 7) ^ (r & 7)) * 16));
}
__device__ __forceinline__ void q_to_tmem(int lane, const uint8_t* scratch, uint32_t taddr) {
  uint32_t out[32];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint4 w = *reinterpret_cast<const uint4*>(scratch + lane * 128 + ((k ^ (lane & 7)) * 16));
    out[4 * k] = w.x;
    out[4 * k + 1] = w.y;
    out[4 * k + 2] = w.z;
    out[4 * k + 3] = w.w;
  }
  tmem_st32(taddr, out);
}

// Split cluster barrier: what this thread wrote before the arrive is visible
// to the other CTAs' threads after their wait.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }

template <int G>
__global__ void __launch_bounds__(kPxThreads, 1) fwd_prefix_kernel(const PrefixParams p,
                                                                   const __grid_constant__ Maps maps) {
  using C = Cfg<G>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* const sbase = smem_raw + (base - raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool score = rank < (uint32_t)G;
  const uint32_t idx = rank % G;                // row tile of the item; CTA 0 of a pair issues its MMAs
  const uint32_t lead = rank - idx, partner = score ? rank + G : rank - G;
  constexpr uint16_t kScoreMask = (1u << G) - 1u, kValueMask = kScoreMask << G, kAllMask = kScoreMask | kValueMask;
  const int item = (int)(blockIdx.x / (2 * G));
  const int sp = item % p.split;
  const long long mt = (long long)(item / p.split) * G + idx;
  const size_t part_at = (size_t)mt * p.split + sp;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sbase + C::kOffAbort);
  auto bar = [&](int i) -> uint32_t { return base + 8u * (uint32_t)i; };
  // one arrival on the leader's barrier
  auto arrive_lead = [&](int i) {
    if (idx == 0) mbar_arrive(bar(i));
    else mbar_arrive_at(mapa_shared(bar(i), lead));
  };
  grid_launch_dependents();  // the own keys' kernel needs nothing from this one

  // keys [tile0 * 64, ...) of the split: whole tiles of the keys in use
  const int used = p.length != nullptr ? min(max(__ldg(p.length), 0), p.keys) : p.keys;
  const int all_tiles = (used + 63) / 64;
  const int tile0 = (int)((long long)all_tiles * sp / p.split);
  const int ntiles = (int)((long long)all_tiles * (sp + 1) / p.split) - tile0;
  const int last_valid = used - (tile0 + ntiles - 1) * 64;  // keys of the item's last tile (64 and more: a full one)
  const bool direct = p.part_num == nullptr;
  const long long row0 = mt * kPxRows;                      // past the rows for the second tile of an odd count

  if (ntiles == 0) {  // the same in all CTAs: nothing to attend to
    for (int r = threadIdx.x; r < kPxRows && row0 + r < p.rows; r += kPxThreads) {
      if (score && direct) {
        p.out_max[row0 + r] = -INFINITY;
        p.out_sum[row0 + r] = 0.f;
      } else if (score) {
        p.part_max[part_at * kPxRows + r] = kNegFltMax;
        p.part_sum[part_at * kPxRows + r] = 0.f;  // the join does not use the numerator then
      }
    }
    if (!score && direct)
      for (int c = threadIdx.x; c < kPxRows * 64; c += kPxThreads)
        if (row0 + (c >> 6) < p.rows)
          reinterpret_cast<uint4*>(p.out + (row0 + (c >> 6)) * kDimLatent)[c & 63] = make_uint4(0, 0, 0, 0);
    return;
  }

  // the softmax warps' chunks of Q are under way while the CTA sets up: group 0
  // takes chunks 0-4, group 1 5-8, the first two through shared memory (in the P
  // staging slots: P of a tile is written after every warp's Q is in TMEM)
  const int q_group = (warp - kSoftWarp0) >> 2;
  const uint32_t q_scratch = C::kOffLocal + (uint32_t)(warp - kSoftWarp0) * 8192u;
  uint4 q_rest[3][8];
  if (score && warp >= kSoftWarp0) {
    const QRows rows(p, row0 + (warp & 3) * 32, lane);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k)
        cp_async_16(base + q_scratch + (uint32_t)i * 4096u + q_place(lane, k), rows.piece(5 * q_group + i, k));
    cp_async_commit();
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (i < 2 || q_group == 0)
#pragma unroll
        for (int k = 0; k < 8; ++k) q_rest[i][k] = __ldg(rows.piece(5 * q_group + 2 + i, k));
  }
  // one barrier per thread (each CTA uses its own part of them)
  if (threadIdx.x < C::kBarCount) mbar_init(bar((int)threadIdx.x), C::bar_count((int)threadIdx.x));
  if (threadIdx.x == 0) *abort_flag = 0;
  fence_barrier_init();
  if (warp == 0) tmem_take<G>(base + C::kOffTmemSlot);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(sbase + C::kOffTmemSlot);
  if (!score && threadIdx.x == 0) {
    for (int s = 0; s < kPSlots; ++s) mbar_arrive_expect_tx(bar(C::kPFull0 + s), kMsgBytes);
    mbar_arrive_expect_tx(bar(C::kFin), kFinBytes);
  }
  __syncwarp();
  // Each role waits for the other CTAs' barriers before it first addresses
  // them, or at its end; Q (and with one CTA a pair, the keys) load without it.
  cluster_arrive();

  bool ok = true;
  if (score) {
    // =============================== score CTAs ===============================
    if (warp == 0) {
      // ---- TMA: part j of tile t into stage t % kKStages; one thread ----
      if (G > 1) cluster_wait();  // loads complete on the leader's barriers
      if (lane == 0) {
        const uint32_t full0 = idx == 0 ? bar(C::kKFull0) : mapa_shared(bar(C::kKFull0), lead);
        auto free_wait = [&](int t, int j) {  // tile t's MMAs have read part j
          return mbar_wait(bar(C::kKFree0 + (t % C::kKStages) * kKParts + j), (uint32_t)(t / C::kKStages) & 1u, abort_flag);
        };
        int t = 0, j = 0;
        for (; t < ntiles; ++t) {
          const int s0 = t % C::kKStages * kKParts;
          const uint32_t stage = base + C::kOffData + (uint32_t)(t % C::kKStages) * C::kKTile;
          for (j = 0; j < kKParts; ++j) {
            if (t >= C::kKStages && !(ok = free_wait(t - C::kKStages, j))) break;
            if (idx == 0) mbar_arrive_expect_tx(bar(C::kKFull0 + s0 + j), (j < 2 ? 4u : 1u) * C::kKBlk * G);
            tma_load_3d<(G > 1)>(stage + (uint32_t)j * 4u * C::kKBlk, j < 2 ? &maps.k : &maps.rope,
                                 (tile0 + t) * 64 + (int)idx * (64 / G), j < 2 ? 4 * j : 0, full0 + 8u * (uint32_t)(s0 + j));
          }
          if (!ok) break;
        }
        if (ok) {  // the last commits arrive in this CTA's memory
          for (int k = max(0, ntiles - C::kKStages); k < ntiles && ok; ++k)
            for (int i = 0; i < kKParts && ok; ++i) ok = free_wait(k, i);
        } else if (idx == 0) {  // loads in flight land before the CTAs' memory goes
          for (int n = max(0, kKParts * (t - C::kKStages) + j); n < kKParts * t + j; ++n)
            mbar_wait_drain(bar(C::kKFull0 + n % (kKParts * C::kKStages)), (uint32_t)(n / (kKParts * C::kKStages)) & 1u);
        }
      }
      __syncwarp();
      if (G == 1) cluster_wait();
    } else if ((warp == 1 || warp == 3) && idx == 0) {
      // ---- QK issuer i: S buffer i <- Q . K^T for tiles g = i mod 2, part by part ----
      const int i = warp >> 1;
      const uint32_t idesc = idesc_bf16(128 * G, 64, false, false);
      ok = wait_warp(bar(C::kQFull), 0u, abort_flag, G > 1);
      tc_fence_after();
      const uint32_t d = tmem + kTmemS + (uint32_t)i * 64u;
      for (int g = i; g < ntiles && ok; g += 2) {
        if (g >= 2 && !(ok = wait_warp(bar(C::kSFree0 + i), (uint32_t)((g >> 1) - 1) & 1u, abort_flag, G > 1))) break;
        const uint32_t st = (uint32_t)g % C::kKStages, s0 = st * kKParts;
        const uint64_t bd = smem_desc(base + C::kOffData + st * C::kKTile, 16, 1024, kLayoutSw128);
#pragma unroll
        for (int part = 0; part < kKParts; ++part) {
          if (!(ok = wait_warp(bar(C::kKFull0 + s0 + part), (uint32_t)(g / C::kKStages) & 1u, abort_flag, G > 1))) break;
          // tiles in turn: two at once would finish together, and the tensor core
          // wait for both S buffers to be read
          if (part == 0 && g > 0 && !(ok = wait_warp(bar(C::kTurn0 + i), (uint32_t)((g - 1) >> 1) & 1u, abort_flag))) break;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int j = 4 * part; j < (part < 2 ? 4 * part + 4 : 9); ++j)
#pragma unroll
              for (int k = 0; k < 4; ++k)  // offsets in the descriptor's 16-byte units; 16 dims are 32 bytes
                mma_ts<G>(d, tmem + kTmemQ + (uint32_t)(j * 4 + k) * 8u, bd + (uint64_t)(j * (C::kKBlk / 16u) + 2 * k), idesc,
                          (j | k) ? 1u : 0u);
            commit_to<G>(bar(C::kKFree0 + s0 + part), kScoreMask);
            if (part == kKParts - 1) {
              commit_to<G>(bar(C::kSFull0 + i), kScoreMask);
              mbar_arrive(bar(C::kTurn0 + (i ^ 1)));
            }
          }
          __syncwarp();
        }
      }
      if (!ok) {
        if (elect_one()) commit_to<G>(bar(C::kDrain0 + i), 1u);  // rank 0: this CTA
        __syncwarp();
        mbar_wait_drain(bar(C::kDrain0 + i), 0u);
      }
      __syncwarp();
      cluster_wait();
    } else if (warp == 2) {
      // ---- P sender: staging slot g % 4 -> the value CTA's P slot g % 4 ----
      const uint32_t r_slot0 = mapa_shared(base + C::kOffSlot, partner);
      const uint32_t r_pfull0 = mapa_shared(bar(C::kPFull0), partner);
      cluster_wait();
      int g = 0;
      for (; g < ntiles; ++g) {
        const uint32_t ls = (uint32_t)g % kLSlots, ps = (uint32_t)g % kPSlots;
        if (!(ok = wait_warp(bar(C::kLFull0 + ls), (uint32_t)(g / kLSlots) & 1u, abort_flag))) break;
        if (g >= kPSlots && !(ok = wait_warp(bar(C::kPDone0 + ps), (uint32_t)(g / kPSlots - 1) & 1u, abort_flag))) break;
        if (lane == 0)
          bulk_copy_to_peer(r_slot0 + ps * kSlotBytes, base + C::kOffLocal + ls * kSlotBytes, kMsgBytes,
                            r_pfull0 + 8u * ps);
        __syncwarp();
      }
      // the value CTAs' last commits arrive in this CTA's memory
      for (int k = max(0, ntiles - kPSlots); k < ntiles && ok; ++k)
        ok = wait_warp(bar(C::kPDone0 + k % kPSlots), (uint32_t)(k / kPSlots) & 1u, abort_flag);
    } else if (warp >= kSoftWarp0) {
      // ---- softmax: one row per thread; group e takes tiles g % 2 == e ----
      const int quad = warp & 3;
      const int e = (warp - kSoftWarp0) >> 2;
      const int row = quad * 32 + lane;
      const uint32_t t_lane = (uint32_t)(quad * 32) << 16;
      const float c = p.scale_log2;
      float* const mpub = reinterpret_cast<float*>(sbase + C::kOffM);
      float* const xch = reinterpret_cast<float*>(sbase + C::kOffX);
      {
        uint8_t* const scratch = sbase + q_scratch;
        const uint32_t tq = tmem + t_lane + kTmemQ + (uint32_t)e * 160u;  // chunk 5 e
        cp_async_wait<0>();
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 2; ++i) q_to_tmem(lane, scratch + i * 4096, tq + (uint32_t)i * 32u);
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          if (i == 2 && e != 0) break;
          uint8_t* const at = scratch + (i & 1) * 4096;
          __syncwarp();  // what was there has been read
#pragma unroll
          for (int k = 0; k < 8; ++k) *reinterpret_cast<uint4*>(at + q_place(lane, k)) = q_rest[i][k];
          __syncwarp();
          q_to_tmem(lane, at, tq + (uint32_t)(2 + i) * 32u);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        cluster_wait();
        if (lane == 0) arrive_lead(C::kQFull);
      }
      float m_w = kNegFltMax, m_true = kNegFltMax, l = 0.f;
      for (int g = e; g < ntiles; g += 2) {
        const uint32_t b = (uint32_t)g % kSBufs;
        if (!(ok = wait_warp(bar(C::kSFull0 + b), (uint32_t)(g / kSBufs) & 1u, abort_flag))) break;
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
        if (lane == 0) arrive_lead(C::kSFree0 + b);
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
          if (!(ok = wait_warp(bar(C::kMReady0 + quad), (uint32_t)(g - 1) & 1u, abort_flag))) break;
          m_prev = mpub[(((g - 1) & 1) * 4 + quad) * 32 + lane];
        }
        const float m_t = ((mx - m_prev) * c > 8.f) ? mx : m_prev;  // lazy rescale threshold 2^8
        mpub[((g & 1) * 4 + quad) * 32 + lane] = m_t;
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(C::kMReady0 + quad));
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
          if (!(ok = wait_warp(bar(C::kPDone0 + gp % kPSlots), (gp / kPSlots) & 1u, abort_flag))) break;
        }
        const uint32_t ls = (uint32_t)g % kLSlots;
        uint8_t* const slot = sbase + C::kOffLocal + ls * kSlotBytes;
        uint8_t* const prow = slot + (uint32_t)(row >> 3) * 1024u + (uint32_t)(row & 7) * 128u;
#pragma unroll
        for (int q = 0; q < 8; ++q)
          *reinterpret_cast<uint4*>(prow + (uint32_t)((q ^ (row & 7)) * 16)) =
              make_uint4(packed[4 * q], packed[4 * q + 1], packed[4 * q + 2], packed[4 * q + 3]);
        *reinterpret_cast<float*>(slot + kAlphaOff + (uint32_t)row * 4u) = alpha;
        if (lane == 0) *reinterpret_cast<uint32_t*>(slot + kFlagOff + (uint32_t)quad * 4u) = flag;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(C::kLFull0 + ls));
      }
      // ---- totals of the two groups ----
      if (ok) {
        float* const mine = xch + (quad * 2 + e) * 96;
        const float* const other = xch + (quad * 2 + (e ^ 1)) * 96;
        mine[lane] = m_w;
        mine[32 + lane] = l;
        mine[64 + lane] = m_true;
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(C::kXchg0 + quad));
        ok = wait_warp(bar(C::kXchg0 + quad), 0u, abort_flag);
        if (ok && e == 0) {
          const float m_o = other[lane], l_o = other[32 + lane];
          const float m_fin = fmaxf(m_w, m_o);
          l = (m_w == m_fin ? l : l * ex2((m_w - m_fin) * c)) + (m_o == m_fin ? l_o : l_o * ex2((m_o - m_fin) * c));
          m_true = fmaxf(m_true, other[64 + lane]);
          const float f = m_true == kNegFltMax ? 1.f : ex2((m_fin - m_true) * c);
          if (row0 + row < p.rows) {
            if (direct) {
              p.out_max[row0 + row] = final_max(m_true, l, p.scale_div);
              p.out_sum[row0 + row] = l * f;
            } else {
              p.part_max[part_at * kPxRows + row] = m_true == kNegFltMax ? kNegFltMax : __fdiv_rn(m_true, p.scale_div);
              p.part_sum[part_at * kPxRows + row] = l * f;
            }
          }
          st_async_b32x2(mapa_shared(base + C::kOffFin, partner) + (uint32_t)row * 8u, mapa_shared(bar(C::kFin), partner),
                         f2u(l), f2u(f));
        }
      }
    } else {
      cluster_wait();
    }
  } else {
    // =============================== value CTAs ===============================
    if (warp == 0) {
      // ---- TMA: this CTA's columns of half n = 2 t + h into slot n % kVSlots; one thread. A last tile with keys
      // missing goes to this CTA's own barriers, for the receiver to clear its end ----
      if (G > 1) cluster_wait();
      if (lane == 0) {
        const uint32_t full0 = idx == 0 ? bar(C::kVFull0) : mapa_shared(bar(C::kVFull0), lead);
        const int ends = last_valid < 64 ? 2 * (ntiles - 1) : 2 * ntiles;
        auto free_wait = [&](int n) {  // half n's MMAs are done
          return mbar_wait(bar(C::kVFree0 + n % C::kVSlots), (uint32_t)(n / C::kVSlots) & 1u, abort_flag);
        };
        int n = 0;
        for (; n < 2 * ntiles; ++n) {
          const uint32_t s = (uint32_t)n % C::kVSlots;
          if (n >= C::kVSlots && !(ok = free_wait(n - C::kVSlots))) break;
          const uint32_t dst = base + C::kOffData + s * C::kVBox;
          const int row = (tile0 + (n >> 1)) * 64, blk = (n & 1) * 4 + (int)idx * (4 / G);
          if (n < ends) {
            if (idx == 0) mbar_arrive_expect_tx(bar(C::kVFull0 + s), C::kVBox * G);
            tma_load_3d<(G > 1)>(dst, &maps.v, row, blk, full0 + 8u * s);
          } else {
            mbar_arrive_expect_tx(bar(C::kVLast0 + (n & 1)), C::kVBox);
            tma_load_3d<false>(dst, &maps.v, row, blk, bar(C::kVLast0 + (n & 1)));
          }
        }
        if (ok) {  // the last commits arrive in this CTA's memory
          for (int k = max(0, 2 * ntiles - C::kVSlots); k < 2 * ntiles && ok; ++k) ok = free_wait(k);
        } else {
          for (int k = max(0, n - C::kVSlots); k < n; ++k) {
            if (k >= ends) mbar_wait_drain(bar(C::kVLast0 + (k & 1)), 0u);
            else if (idx == 0) mbar_wait_drain(bar(C::kVFull0 + k % C::kVSlots), (uint32_t)(k / C::kVSlots) & 1u);
          }
        }
      }
      __syncwarp();
      if (G == 1) cluster_wait();
    } else if ((warp == 1 || warp == 3) && idx == 0) {
      // ---- PV issuer h: O[:, 256 h .. 256 h + 255] += P . V ----
      const int h = warp >> 1;
      cluster_wait();
      const uint32_t idesc = idesc_bf16(128 * G, 256, false, true);
      for (int g = 0; g < ntiles; ++g) {
        const uint32_t s = (uint32_t)g % kPSlots;
        if (!(ok = wait_warp(bar(C::kPReady0 + s), (uint32_t)(g / kPSlots) & 1u, abort_flag, true))) break;
        const int n = 2 * g + h;
        const uint32_t vs = (uint32_t)n % C::kVSlots;
        if ((g + 1 < ntiles || last_valid >= 64) &&
            !(ok = wait_warp(bar(C::kVFull0 + vs), (uint32_t)(n / C::kVSlots) & 1u, abort_flag, G > 1)))
          break;
        const uint32_t slot = base + C::kOffSlot + s * kSlotBytes, vslot = base + C::kOffData + vs * C::kVBox;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            mma_ss<G>(tmem + kTmemO + h * 256, smem_desc(slot + j * 32, 16, 1024, kLayoutSw128),
                      smem_desc(vslot + j * 2048, kBlk, 1024, kLayoutSw128), idesc, (g | j) ? 1u : 0u);
          commit_to<G>(bar(C::kVFree0 + vs), kValueMask);
          commit_to<G>(bar(C::kPDone0 + s), kAllMask);
        }
        __syncwarp();
      }
      if (!ok) {
        if (elect_one()) commit_to<G>(bar(C::kDrain0 + h), (uint16_t)(1u << G));  // rank G: this CTA
        __syncwarp();
        mbar_wait_drain(bar(C::kDrain0 + h), 0u);
      }
    } else if (warp == 2) {
      // ---- receiver of P ----
      volatile uint32_t* const req = reinterpret_cast<volatile uint32_t*>(sbase + C::kOffReq);
      cluster_wait();
      uint32_t nresc = 0;
      for (int g = 0; g < ntiles; ++g) {
        const uint32_t s = (uint32_t)g % kPSlots;
        if (!(ok = wait_warp(bar(C::kPFull0 + s), (uint32_t)(g / kPSlots) & 1u, abort_flag, true))) break;
        if (lane == 0 && g + kPSlots < ntiles) mbar_arrive_expect_tx(bar(C::kPFull0 + s), kMsgBytes);  // its next message
        __syncwarp();
        const volatile uint32_t* fl = reinterpret_cast<const volatile uint32_t*>(sbase + C::kOffSlot + s * kSlotBytes + kFlagOff);
        if ((fl[0] | fl[1] | fl[2] | fl[3]) != 0u) {
          if (lane == 0) {
            *req = (uint32_t)g;
            mbar_arrive(bar(C::kReq));
          }
          __syncwarp();
          if (!(ok = wait_warp(bar(C::kReqDone), nresc & 1u, abort_flag))) break;
          ++nresc;
          tc_fence_after();  // the rescaled O goes on to the issuers' MMAs
          tc_fence_before();
        }
        if (g + 1 == ntiles && last_valid < 64) {
          // rows behind the last key: weight 0, but 0 x NaN of a cache row never written would not be 0
          for (int h = 0; h < 2 && ok; ++h) {
            if (!(ok = wait_warp(bar(C::kVLast0 + h), 0u, abort_flag))) break;
            uint8_t* const vslot = sbase + C::kOffData + (uint32_t)((2 * g + h) % C::kVSlots) * C::kVBox;
            constexpr int kPieces = 8 * (4 / G);  // 16-byte pieces of a key's row here
            for (int i = lane; i < (64 - last_valid) * kPieces; i += 32) {
              const int r = last_valid + i / kPieces, q = i % kPieces;
              *reinterpret_cast<uint4*>(vslot + (uint32_t)(q >> 3) * kBlk + (uint32_t)r * 128u + (uint32_t)(q & 7) * 16u) =
                  make_uint4(0, 0, 0, 0);
            }
          }
          if (!ok) break;
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) arrive_lead(C::kPReady0 + s);
      }
      if (ok && lane == 0) {
        *req = kReqEnd;
        mbar_arrive(bar(C::kReq));
      }
      __syncwarp();
    } else if (warp >= kSoftWarp0) {
      // ---- rescale requests, then the epilogue: half `part` of the columns of 32 rows ----
      const int quad = warp & 3, part = (warp - kSoftWarp0) >> 2;
      cluster_wait();
      const int row = quad * 32 + lane;
      const uint32_t t_o = tmem + ((uint32_t)(quad * 32) << 16) + kTmemO + (uint32_t)part * 256u;
      const volatile uint32_t* const req = reinterpret_cast<const volatile uint32_t*>(sbase + C::kOffReq);
      auto pv_done = [&](int g) { return wait_warp(bar(C::kPDone0 + g % kPSlots), (uint32_t)(g / kPSlots) & 1u, abort_flag); };
      for (uint32_t nreq = 0;; ++nreq) {
        if (!(ok = wait_warp(bar(C::kReq), nreq & 1u, abort_flag))) break;
        const uint32_t g = *req;
        if (g == kReqEnd) break;
        const uint8_t* slot = sbase + C::kOffSlot + (g % kPSlots) * kSlotBytes;
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
        if (lane == 0) mbar_arrive(bar(C::kReqDone));
      }
      if (ok && (ok = wait_warp(bar(C::kFin), 0u, abort_flag, true)) && (ok = pv_done(ntiles - 1))) {
        const volatile float* lf = reinterpret_cast<const volatile float*>(sbase + C::kOffFin + row * 8);
        const float l = lf[0], f = lf[1];
        tc_fence_after();
        const long long grow = row0 + row;
        const bool live = grow < p.rows;
        const bool any = row0 + quad * 32 < p.rows;  // the warp has a row
        if (direct) {
          const float rl = l > 0.f || l != l ? __frcp_rn(l) : 0.f;
          __nv_bfloat16* const dst = p.out + (size_t)(grow & ~1LL) * kDimLatent + part * 256;
          const bool wide = (reinterpret_cast<uintptr_t>(p.out) & 31u) == 0;
#pragma unroll 1
          for (int cb = 0; cb < 256 && any; cb += 32) {
            uint32_t o[32];
            tmem_ld32(t_o + (uint32_t)cb, o);
            tmem_wait_ld_regs32(o);
            uint32_t a[8], b[8];
            pack_bf16_row32_paired(o, rl, a, b);
            if (live) store_bf16_row32_paired(dst + cb, kDimLatent, a, b, wide);  // rows is even: pairs are whole
          }
        } else {
          // [64 groups of 8 columns][128 rows][8]: a store instruction writes 1 KB in a row
          float* const dst = p.part_num + (part_at * 64 + part * 32) * (kPxRows * 8) + row * 8;
#pragma unroll 1
          for (int cb = 0; cb < 256 && any; cb += 64) {
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
    tmem_give<G>(tmem);
  }
}

// Join of a row's prefix partials and its own-key partials: m = max m_i,
// out = sum_i e^(m_i - m) n_i / sum_i e^(m_i - m) l_i. A block takes 32 rows
// (lane = row) and 64 columns (8 a warp) and shares its rows' (m, l) in shared
// memory. Bound by the partials' 2 KB a row and part, and with few rows by
// latency: a thread's first four parts are under way before the weights are
// known (8192 rows of 3 parts 20 -> 15 us from DRAM; eight in flight cost
// occupancy, 21 us). A part without keys (sum 0) is left out: nothing is written
// to its numerator then. Every other part counts, whatever its weight: the
// maximum of a part whose scores are all NaN says nothing, and its NaN sum has
// to reach the row.
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
      if (ml.y != 0.f) {
        const float w = expf(ml.x - top);
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
    p.out_max[r] = total > 0.f ? top : -INFINITY;  // -inf beside a NaN sum, as final_max gives
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
// box_blocks x box_rows x 64.
bool encode(CUtensorMap* map, const void* ptr, long long rows, int blocks, int box_rows, int box_blocks) {
  const EncodeFn fn = encode_fn();
  if (fn == nullptr) return false;
  const cuuint64_t dims[3] = {64, (cuuint64_t)rows, (cuuint64_t)blocks};
  const cuuint64_t strides[2] = {(cuuint64_t)blocks * 128u, 128u};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, (cuuint32_t)box_blocks};
  const cuuint32_t ones[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(ptr), dims, strides, box, ones,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int G>
bool launch_config(cudaLaunchConfig_t* cfg, cudaLaunchAttribute* attr, unsigned ctas, cudaStream_t stream) {
  // once per device: the attribute belongs to the device's context
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if ((ready.load(std::memory_order_relaxed) & bit) == 0) {
    if (cudaFuncSetAttribute(fwd_prefix_kernel<G>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)Cfg<G>::kSmemBytes) != cudaSuccess)
      return false;
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  attr->id = cudaLaunchAttributeClusterDimension;
  attr->val.clusterDim.x = 2 * G;
  attr->val.clusterDim.y = 1;
  attr->val.clusterDim.z = 1;
  *cfg = cudaLaunchConfig_t{};
  cfg->gridDim = dim3(ctas, 1, 1);
  cfg->blockDim = dim3(kPxThreads, 1, 1);
  cfg->dynamicSmemBytes = Cfg<G>::kSmemBytes;
  cfg->stream = stream;
  cfg->attrs = attr;
  cfg->numAttrs = 1;
  return true;
}

template <int G>
int max_clusters() {
  static std::atomic<int> cached{-1};
  int n = cached.load(std::memory_order_relaxed);
  if (n > 0) return n;
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr;
  if (!launch_config<G>(&cfg, &attr, 148, nullptr) ||
      cudaOccupancyMaxActiveClusters(&n, fwd_prefix_kernel<G>, &cfg) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    return -1;
  }
  cached.store(n, std::memory_order_relaxed);
  return n;
}

template <int G>
cudaError_t launch(const PrefixParams& p, const void* kv, const void* k_rope, cudaStream_t stream) {
  Maps maps;
  if (!encode(&maps.k, kv, p.keys, 8, 64 / G, 4) || !encode(&maps.v, kv, p.keys, 8, 64, 4 / G) ||
      !encode(&maps.rope, k_rope, p.keys, 1, 64 / G, 1))
    return cudaErrorInvalidValue;
  const long long tiles = (p.rows + kPxRows - 1) / kPxRows;
  const long long items = (tiles + G - 1) / G * p.split;
  if (items <= 0 || 2 * G * items > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr;
  if (!launch_config<G>(&cfg, &attr, (unsigned)(2 * G * items), stream)) return cudaErrorInvalidConfiguration;
  return cudaLaunchKernelEx(&cfg, fwd_prefix_kernel<G>, p, maps);
}

}  // namespace

int prefix_max_clusters(int group) { return group == 2 ? max_clusters<2>() : max_clusters<1>(); }

cudaError_t launch_fwd_prefix(const PrefixParams& p, const void* kv, const void* k_rope, cudaStream_t stream) {
  return p.group == 2 ? launch<2>(p, kv, k_rope, stream) : launch<1>(p, kv, k_rope, stream);
}

cudaError_t launch_prefix_join(const JoinParams& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr;
  // Its blocks wait themselves: beside the prefix kernel where there are no own
  // keys; the own keys' kernel lets them start only at its own end.
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
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
