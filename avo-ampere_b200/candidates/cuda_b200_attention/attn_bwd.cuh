// Gradient of attention for sm_100a (B200), head_dim 128, bf16 in and out.
//
// With S = scale * Q K^T, P = exp(S - LSE) (0 where the mask hides the key), dP = dO V^T and
// delta_i = sum_d dO_id O_id:
//     dS = P * (dP - delta),  dQ = scale * dS K,  dK = scale * dS^T Q,  dV = P^T dO,
// dK and dV summed over the query heads that share a key/value head.  The probabilities are
// recomputed from Q, K and the LSE the forward saved.
//
// Three launches, and a fourth (join_kernel) where work is split.  stats_kernel writes
// -LSE*log2(e) and -delta per query row.  Then one kernel template runs twice over 128 x 128
// tiles, each time with one side of the tile stationary and the other streamed through shared
// memory:
//
//             rows (M)   stationary X1, X2   streamed Y1, Y2   accumulators in TMEM
//   dK/dV     keys       K, V                Q, dO             dK += dS^T Q, dV += P^T dO
//   dQ        queries    Q, dO               K, V              dQ += dS K
//
//   T1 = X1 Y1^T (S or S^T), T2 = X2 Y2^T (dP or dP^T); the softmax warps turn them into P
//   and dS, bf16, in TMEM, where they are the A operand of the accumulating MMAs.
//
// Two passes recompute S and dP: 7 products per tile pair instead of the 5 that one pass
// needs.  In exchange dQ is not accumulated across CTAs: no atomics (the result does not
// depend on the order in which CTAs run), no fp32 dQ in memory, and neither P nor dS ever
// leaves TMEM.  Per tile the tensor pipe needs 2048 (dK/dV) and 1536 (dQ) cycles, and the
// 512 softmax threads' work on it overlaps, phase against phase:
//
//   dK/dV:  tensor   | dV_n  S_{n+1} | dK_n  dP_{n+1} | dV_{n+1} ...
//           softmax  | dS_n from dP_n | P_{n+1} from S_{n+1} | ...
//   dQ:     tensor   | S_{n+1} | dP_{n+1} | dQ_n | ...
//           softmax  | P_n from S_n | dS_n from dP_n | P_{n+1} ...
//
// In dK/dV, TMEM holds T1, T2 and two accumulators, so P and dS replace T1 and T2 in place
// and a T is only recomputed once the MMA that reads its P or dS has been issued.  dQ has one
// accumulator; the free columns hold dS and Q itself (as the A operand of S: one tile less
// in shared memory and 32 KB less to read from it per tile, which leaves room for a fourth
// K slot), so S_{n+1} and dP_{n+1} start as soon as S_n and dP_n are in registers.
//
// Sums are fp32 in TMEM; P and dS are rounded once to bf16 (the type of the tensor cores'
// operands: at most half a step, 2^-8 of each value), the gradients once at the end.
//
// What bounds it, measured on B200.  B4 H16 S4096 back to back: 1508 us, 1276 TFLOPS of the
// seven products, 93 % of cuBLAS's sustained rate, at the chip's power limit (1.40 GHz); a tile
// pair takes 2408 (dK/dV) and 1844 (dQ) cycles.  An item's start and end cost 2.4 and 1.3 us more
// than its tiles (the last accumulators are read out before the next item adds to them): 18 % of
// the time at B8 H16 S2048 causal, where an item has 8.5 tiles.  Small calls: 11.5 us at B1 H4
// S512, the latency of 4 tiles in either pass.
//
// Roles (768 threads): warps 0-15 softmax (four warpgroups, 32 of a tile's 128 columns each),
// warps 16-19 the epilogue (an item's accumulators to memory, and Q of the next item to TMEM,
// while the tile loop runs), warp 20 TMA producer, warp 21 MMA issuer, warp 22 waiter: the
// issuer waits on hardware named barriers only, because a shared-memory read by the issuing
// thread drains its queued MMAs first.  Every wait is bounded by the watchdog, and after an
// abort every role still takes its fixed number of barrier rounds, so no CTA is left waiting.
#pragma once

#include <cuda_bf16.h>

#include <climits>

#include "attn_fwd.cuh"

namespace avo_b200 {
namespace bwd {

constexpr int kTile = 128;
constexpr int kSoftmaxThreads = 512;
constexpr int kEpiWarp = 16;
constexpr int kProducerWarp = 20;
constexpr int kIssuerWarp = 21;
constexpr int kWaiterWarp = 22;
constexpr int kBwdThreads = 768;
// Launched at 80 registers per thread (768 x 80 = 61440); after the split 512 x 88 + 128 x 80
// + 128 x 48 = 61440.
constexpr uint32_t kBwdRegsLaunch = 80;
constexpr uint32_t kBwdRegsSoftmax = 88;
constexpr uint32_t kBwdRegsEpi = 80;
constexpr uint32_t kBwdRegsOther = 48;
static_assert(kSoftmaxThreads * kBwdRegsSoftmax + 128 * kBwdRegsEpi + 128 * kBwdRegsOther <= kBwdThreads * kBwdRegsLaunch,
              "register split");

// A wait that lasts as long as an item of `tiles` tiles: one lane polls, asleep in between,
// so that it takes no issue slots and no shared-memory bandwidth from the tile loop.  Each
// of the item's tiles has a watchdog of its own, so their sum bounds this wait.
__device__ __forceinline__ bool wait_item(uint32_t bar, uint32_t parity, int tiles, const Watch& w, int lane) {
  bool ok = true;
  if (lane == 0 && !mbar_try_wait(bar, parity)) {
    const uint64_t t0 = global_timer_ns();
    while (!mbar_try_wait_sleep(bar, parity, 20000)) {
      ok = !*w.abort;
      if (ok && (global_timer_ns() - t0) / (static_cast<uint64_t>(tiles) + 2) > w.limit_ns) {
        *w.abort = 1;
        if (w.status != nullptr) atomicOr(w.status, kStatusWatchdog);
        ok = false;
      }
      if (!ok) break;
    }
  }
  return __all_sync(0xffffffffu, ok);
}

// Named barriers, all synced by the issuer.  Those with two ids alternate (by tile, or by
// item): an arrival is then never counted to a round that the issuer has not reached, also
// after an abort, when a warp no longer waits for the MMAs that order the rounds.
//   3             first tile's operands loaded (waiter)
//   dK/dV: 4/7, 5/8  halves of P in TMEM (softmax warps; 5/8: and the waiter, next T1's operand)
//          6/9       dS in TMEM (softmax, and the waiter: next T2's operand)
//          10/11, 12/13  accumulator 1 / 2 read out (epilogue warps)
//   dQ:    4/7, 5/8  T1 / T2 in registers (softmax, and the waiter: next T1's / T2's operand)
//          6/9       dS in TMEM (softmax)
//          10/11     accumulator read out, 12/13 next item's Q in TMEM (epilogue warps)
constexpr uint32_t kBarLoaded = 3;
enum : uint32_t { kRoundP0 = 4, kRoundP1 = 5, kRoundT1Read = 4, kRoundT2Read = 5, kRoundDs = 6 };
__device__ __forceinline__ uint32_t bar_tile(uint32_t round, uint32_t tile) { return round + (tile & 1) * 3; }
__device__ __forceinline__ uint32_t bar_acc1(uint32_t item) { return 10 + (item & 1); }
__device__ __forceinline__ uint32_t bar_acc2(uint32_t item) { return 12 + (item & 1); }
__device__ __forceinline__ uint32_t bar_x1(uint32_t item) { return 12 + (item & 1); }
constexpr uint32_t kHalfThreads = kSoftmaxThreads + 32;   // softmax and issuer
constexpr uint32_t kTileThreads = kSoftmaxThreads + 64;   // softmax, waiter and issuer
template <bool kDq>
constexpr uint32_t kDsThreads = kDq ? kHalfThreads : kTileThreads;
constexpr uint32_t kEpiThreads = 128 + 32;                // epilogue and issuer

// Shared memory: X1 (dK/dV only), X2, the Y1 slots, two Y2 slots, statistics (dK/dV only).
// Y1 is used by T1 and by the last MMA of its tile.  With two Y1 slots in dK/dV a tile's load
// could only start 1024 tensor cycles before its use, about the latency of a 32 KB load.
constexpr int kY2 = 2;
template <bool kDq>
struct Smem {
  static constexpr int kY1 = kDq ? 4 : 3;
  static constexpr int kX1 = 0;
  static constexpr int kX2 = kDq ? 0 : kTileBytes;
  static constexpr int kY1At = kX2 + kTileBytes;
  static constexpr int kY2At = kY1At + kY1 * kTileBytes;
  static_assert(kY2At + kY2 * kTileBytes == 7 * kTileBytes, "both passes fill seven tiles");
};
constexpr int kSmStat = 7 * kTileBytes;  // two slots of [-LSE*log2 e | -delta], 128 floats each
constexpr int kStatBytes = 2 * kTile * 4;
constexpr int kSmBars = kSmStat + 2 * kStatBytes;
// mbarriers.  The issuer commits after T1 and after T2 of a tile, and these commits also tell
// the producer that the MMAs issued before them are done with their operands (a commit takes
// about 50 cycles of the issuer's time).  dQ's Y1 slots and dK/dV's Y2 slots have a commit of
// their own: with T1's, 512 cycles later, the next load into the slot came too late.
// T1_FULL and T2_FULL are pairs, used by even and odd tiles, so that no wait can miss a phase.
enum : int {
  B_X1_FULL = 0,
  B_X1_DONE = B_X1_FULL,  // dQ: the item's last S is done with Q in TMEM
  B_X2_FULL,
  B_Y1_FULL,
  B_Y1_EMPTY = B_Y1_FULL + 4,
  B_Y2_FULL = B_Y1_EMPTY + 4,
  B_Y2_EMPTY = B_Y2_FULL + kY2,
  B_T1_FULL = B_Y2_EMPTY + kY2,
  B_T2_FULL = B_T1_FULL + 2,
  B_ACC1 = B_T2_FULL + 2,
  B_ACC2,
  B_STAT,
  B_DRAINED = B_STAT + 2,
  B_COUNT
};
constexpr int kSmTmem = kSmBars + B_COUNT * 8;
constexpr int kSmAbort = kSmTmem + 4;
constexpr int kSmSlot = kSmAbort + 4;  // this CTA's place in the order of items
constexpr int kBwdSmemBytes = (kSmSlot + 4 + 15) / 16 * 16;
static_assert(kBwdSmemBytes <= 227 * 1024, "shared memory budget");

constexpr int kMaxClaims = 256;  // multiprocessors, at most, whose CTAs claim a place

// TMEM columns: T1 | T2 | accumulator 1 | accumulator 2 (dK/dV) or dS and Q (dQ).
constexpr uint32_t kColT1 = 0, kColT2 = 128, kColAcc1 = 256, kColAcc2 = 384;
constexpr uint32_t kColDs = 384, kColX1 = 448;

struct BwdParams {
  const float* stats;  // [num_q_heads][nq][2][128]: -LSE*log2(e), -delta
  const void* x1;      // dQ: Q, [q_heads, seq_q, 128]
  void* g1;            // dK or dQ
  void* g2;            // dV, or null
  int* status;
  unsigned long long watchdog_ns;
  int seq_q, seq_kv;
  int nq, nkv;             // 128-row tiles of queries and of keys
  int q_heads, kv_heads;   // batch * heads
  int group;               // query heads per key/value head
  int causal;
  int offset;              // causal: key j is visible to query i iff j <= i + offset
  float scale, scale_log2;
  uint32_t* claims;        // null (place = CTA number), or gridDim.x zeros: places taken
  int test_skip_load;
  // An item is a stationary tile; with split > 1 it is cut into that many pieces along the
  // streamed tiles, each a unit of its own whose sums go to part1 / part2 in fp32
  // ([split][heads][rows][128]), for join_kernel to add.
  uint32_t split;
  unsigned long long split_magic;
  float* part1;
  float* part2;
  uint32_t item_count;     // units, or pairs, of this launch
  uint32_t item_div;       // what an item's number is divided by: heads (causal), tiles or pairs of them
  unsigned long long item_magic;
};

// w / div: with magic = ceil(2^64 / div) the high half of w * magic is exact for every 32-bit
// w (the excess of magic is below 1, its product below 2^-32 of a step).
__device__ __forceinline__ uint32_t div_by(uint32_t w, uint32_t div, unsigned long long magic) {
  return div == 1 ? w : static_cast<uint32_t>(__umul64hi(w, magic));
}

// The order of the items, and what the kernel is compiled for.  Whole items without a mask, or
// with one and equal lengths, are simpler than the general case, and the softmax warps, short
// of registers, gain by that (measured on B200, compiled for all cases / for its own: B4 H16
// S4096 1547 / 1528 us; causal B8 H16 S2048, in pairs in either, 545 / 520).
//   kAny      waves over the grid in alternating directions.  Causal items are of different
//             lengths: longest first, the same tile of all heads before the next tile.
//   kEqual    (no mask, whole items) the same, heads one after the other.
//   kLongest  (causal, equal lengths, whole items) as kAny.
//   kPairs    (the same) heads one after the other, and each CTA takes the first and the last
//             tile of a head, or the second and the last but one, and so on, which together are
//             as long as any other pair.
enum Order : int { kAny, kEqual, kLongest, kPairs };

// One CTA's units in order (a stationary tile of one head, or a piece of its work).
template <bool kDq, Order kOrder>
struct Items {
  const BwdParams& p;
  uint32_t r = 0;
  int head, tile;  // stationary head and tile
  int t0;          // first streamed tile that the item needs
  int n;           // streamed tiles of this unit (dK/dV: over the whole group of heads)
  int skip;        // of the item's tiles, those of earlier pieces
  int piece;
  const volatile uint32_t* slot;
  __device__ Items(const BwdParams& params, const volatile uint32_t* place) : p(params), slot(place) {}
  // The next item that has tiles.
  __device__ bool next_busy() {
    do {
      if (!next()) return false;
    } while (n == 0);
    return true;
  }
  __device__ bool next() {
    const uint32_t grid = gridDim.x, cta = *slot;
    while (true) {
      if constexpr (kOrder == kPairs) {
        const unsigned long long at = static_cast<unsigned long long>(r >> 1) * grid + cta;
        if (at >= p.item_count) return false;
        const uint32_t quotient = div_by(static_cast<uint32_t>(at), p.item_div, p.item_magic);
        head = static_cast<int>(quotient);
        tile = static_cast<int>(static_cast<uint32_t>(at) - quotient * p.item_div);
        if (r++ & 1) {
          const int partner = (kDq ? p.nq : p.nkv) - 1 - tile;
          if (partner == tile) continue;  // the middle tile
          tile = partner;
        }
        piece = 0;
      } else {
        const unsigned long long base = static_cast<unsigned long long>(r) * grid;
        if (base >= p.item_count) return false;
        const uint32_t unit = static_cast<uint32_t>(base) + ((r & 1) ? grid - 1 - cta : cta);
        ++r;
        if (unit >= p.item_count) continue;
        const uint32_t w = kOrder == kAny ? div_by(unit, p.split, p.split_magic) : unit;
        piece = kOrder == kAny ? static_cast<int>(unit - w * p.split) : 0;
        const uint32_t quotient = div_by(w, p.item_div, p.item_magic);
        const int rest = static_cast<int>(w - quotient * p.item_div);
        if (kOrder == kLongest || (kOrder == kAny && p.causal)) {
          head = rest;
          tile = kDq ? p.nq - 1 - static_cast<int>(quotient) : static_cast<int>(quotient);
        } else {
          head = static_cast<int>(quotient);
          tile = rest;
        }
      }
      t0 = 0;
      skip = 0;
      if constexpr (kOrder >= kLongest) {
        if (!kDq) t0 = tile;
        n = kDq ? tile + 1 : (p.nq - tile) * p.group;
        return true;
      }
      if constexpr (kOrder == kEqual) {
        n = kDq ? p.nkv : p.nq * p.group;
        return true;
      }
      if (kDq) {
        n = p.nkv;
        if (p.causal) {
          const int end = min(tile * kTile + kTile, p.seq_q) + p.offset;  // keys the last row sees
          n = min(p.nkv, (max(end, 0) + kTile - 1) >> 7);
        }
      } else {
        // The tile of the first query that sees the tile's first key.  The bounds by nq never
        // bind: offset is seq_kv - seq_q, so the last query sees every key.  They stay for what
        // the compiler makes of them, which without them keeps more of this instance's
        // registers in memory (measured on B200, with / without: B1 H16 Hkv2 Q777 KV5003 104.4 /
        // 106.3 us, B1 H4 Hkv2 Q300 KV900 20.1 / 20.7, B1 H8 Hkv2 S2048 39.6 / 39.9, causal).
        if (p.causal) t0 = min(max(0, tile * kTile - p.offset) >> 7, p.nq);
        if (p.causal && tile * kTile - p.offset >= p.seq_q) t0 = p.nq;
        n = (p.nq - t0) * p.group;
      }
      if (p.split > 1) {
        const uint32_t all = static_cast<uint32_t>(n), pieces = p.split, at = static_cast<uint32_t>(piece);
        skip = static_cast<int>(div_by(all * at, pieces, p.split_magic));
        n = static_cast<int>(div_by(all * (at + 1), pieces, p.split_magic)) - skip;
      }
      return true;
    }
  }
};

// The tiles of a CTA's items as one sequence (items without tiles are skipped).
template <bool kDq, Order kOrder>
struct Tiles {
  Items<kDq, kOrder> items;
  int left = 0;   // tiles of the item still to come
  int t, y_head;  // current streamed tile and its head
  bool first, last;
  __device__ Tiles(const BwdParams& params, const volatile uint32_t* place) : items(params, place) {}
  __device__ bool next() {
    first = false;
    if (left == 0) {
      if (!items.next_busy()) return false;
      left = items.n;
      first = true;
      t = items.t0 + items.skip;
      y_head = kDq ? items.head / items.p.group : items.head * items.p.group;
      if (!kDq && kOrder == kAny && items.skip > 0) {
        const int per_head = items.p.nq - items.t0;
        const int heads = items.skip / per_head;
        y_head += heads;
        t -= heads * per_head;
      }
    } else {
      ++t;
      if (!kDq && t == items.p.nq) {
        t = items.t0;
        ++y_head;
      }
    }
    --left;
    last = left == 0;
    return true;
  }
};

// T = X Y^T for one 128 x 128 tile, both operands K-major.
__device__ __forceinline__ void issue_xy(uint32_t d_tmem, uint32_t x_lo, uint32_t y_lo) {
  issue_qk(d_tmem, x_lo, y_lo, kDescHiSw128);
}

// The same with X in TMEM.
__device__ __forceinline__ void issue_xy_tmem(uint32_t d_tmem, uint32_t x_tmem, uint32_t y_lo) {
  constexpr uint32_t idesc = idesc_bf16_f32(kTile, kTile, 0, 0);
#pragma unroll
  for (int kk = 0; kk < 8; ++kk)
    mma_ts_lo(d_tmem, x_tmem + kk * 8, y_lo + (((kk >> 2) * kHalfBytes + (kk & 3) * 32) >> 4), kDescHiSw128, idesc,
              kk > 0 ? 1u : 0u);
}

// acc (+)= A Y over 64 of the 128 streamed rows: A (P or dS, bf16) from TMEM, Y from shared
// memory as an MN-major operand.  Each softmax warpgroup holds 16 columns of either half; in
// dK/dV its values replace the scores at the place they came from, in dQ they lie packed.
template <bool kPacked>
__device__ __forceinline__ void issue_acc_half(uint32_t d_tmem, uint32_t a_tmem, uint32_t y_lo, int half,
                                               uint32_t accumulate) {
  constexpr uint32_t idesc = idesc_bf16_f32(kTile, kHeadDim, 0, 1);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int kk = half * 4 + q;
    mma_ts_lo(d_tmem, a_tmem + (kPacked ? kk * 8 : kk * 16), y_lo + ((kk * 16 * 128) >> 4),
              kDescHiSw128, idesc, accumulate | (kk > 0 ? 1u : 0u));
  }
}

template <bool kPacked>
__device__ __forceinline__ void issue_acc(uint32_t d_tmem, uint32_t a_tmem, uint32_t y_lo, uint32_t accumulate) {
  issue_acc_half<kPacked>(d_tmem, a_tmem, y_lo, 0, accumulate);
  issue_acc_half<kPacked>(d_tmem, a_tmem, y_lo, 1, accumulate);
}

constexpr int kEmu = 2;

// 2^x for pair number `i` of a chunk: kOf8 of every 8 pairs on the FMA pipe (results below
// 2^-125 become 0: a hidden key's P is exactly 0 on both paths), the others on the MUFU unit.
template <int kOf8>
__device__ __forceinline__ uint64_t exp2_pair(int i, uint64_t x2) {
  float x0, x1, p0, p1;
  f2_unpack(x2, x0, x1);
  if ((i & 7) < kOf8) {
    exp2_poly_x2(x2, p0, p1);
    p0 = x0 < -125.f ? 0.f : p0;
    p1 = x1 < -125.f ? 0.f : p1;
  } else {
    p0 = ex2_approx(x0);
    p1 = ex2_approx(x1);
  }
  return f2_pack(p0, p1);
}

__device__ __forceinline__ uint32_t pack_pair(uint64_t v) {
  float a, b;
  f2_unpack(v, a, b);
  return pack_bf16x2(a, b);
}

template <bool kDq, Order kOrder>
__global__ void __launch_bounds__(kBwdThreads, 1)
    attn_bwd_kernel(const __grid_constant__ CUtensorMap tm_x1, const __grid_constant__ CUtensorMap tm_x2,
                    const __grid_constant__ CUtensorMap tm_y1, const __grid_constant__ CUtensorMap tm_y2,
                    const __grid_constant__ BwdParams p) {
  using Sm = Smem<kDq>;
  using Items = bwd::Items<kDq, kOrder>;
  using Tiles = bwd::Tiles<kDq, kOrder>;
  constexpr int kY1 = Sm::kY1;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_addr(smem);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  auto bar = [&](int idx) -> uint32_t { return sbase + kSmBars + idx * 8; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kSmAbort);
  volatile uint32_t* slot = reinterpret_cast<volatile uint32_t*>(smem + kSmSlot);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kSmTmem);
  const Watch watch{abort_flag, p.status, p.watchdog_ns};

  // The swizzled tiles need a 1024-byte aligned base, and there is no room to align it here.
  if ((sbase & 1023u) != 0) {
    if (threadIdx.x == 0 && p.status != nullptr) atomicOr(p.status, kStatusWatchdog);
    return;
  }
  if (threadIdx.x == 0) {
    for (int b = 0; b < B_COUNT; ++b) mbar_init(bar(b), 1);
    *abort_flag = 0;
    *slot = blockIdx.x;
    fence_mbarrier_init();
  }
  if (warp == kProducerWarp && lane == 0) {
    prefetch_tensormap(&tm_x1);
    prefetch_tensormap(&tm_x2);
    prefetch_tensormap(&tm_y1);
    prefetch_tensormap(&tm_y2);
  }
  if (warp == kIssuerWarp) {
    tmem_alloc(smem_addr(tmem_slot), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // The dK/dV launch follows stats_kernel and waits for it here.  The dQ launch follows the
  // dK/dV launch, reads nothing that it writes, and can only start once all CTAs of that
  // launch have passed this wait; it runs on the multiprocessors that launch leaves free, or
  // is done with, and its last CTA waits for it at the end.
  if (!kDq) {
    grid_dependency_wait();
    grid_launch_dependents();
  }
  // With a unit for every multiprocessor, CTAs take their place in the order of items by
  // multiprocessor (the next free one, should two CTAs ask for the same), and dQ counts from
  // the other end.  Then a multiprocessor that has one item more of dK/dV has the fewest of dQ, and the two of a pair
  // (a TPC) change from one pass to the other at the same time: while they run different
  // kernels, both take up to twice as long (the pair seems to share its instruction cache).
  // Measured on B200, B1 H16 S4096: both passes one after the other 391 to 413 us, at once
  // without such places 411 to 447, with them 335 to 381.
  if (p.claims != nullptr) {
    if (threadIdx.x == 0) {
      const uint32_t grid = gridDim.x;
      uint32_t s = sm_id() % grid;
      for (uint32_t i = 0; i < grid && atomicExch(p.claims + s, 1u) != 0u; ++i) s = s + 1 == grid ? 0 : s + 1;
      *slot = kDq ? grid - 1 - s : s;
    }
    __syncthreads();
  }

  if (warp < kEpiWarp) {
    regs_increase<kBwdRegsSoftmax>();
    // ------------------------------------------------------------ softmax
    // Each warpgroup takes 16 columns of either half of the tile: [16 wg, 16 wg + 16) and
    // 64 further on.
    const int wg = warp >> 2;
    const int wq = warp & 3;
    const int row = threadIdx.x & 127;
    const uint32_t tBase = tmem + (static_cast<uint32_t>(wq * 32) << 16) + wg * 16;
    const uint64_t scale2 = f2_pack(p.scale_log2, p.scale_log2);
    const bool causal = kOrder >= kLongest || (kOrder == kAny && p.causal);
    const int offset = kOrder >= kLongest ? 0 : p.offset;
    uint32_t n = 0;
    float neg_lse = 0.f, neg_delta = 0.f;
    Tiles it(p, slot);
    // The barrier rounds of a tile from round `from` on, blocking: after an abort a warp
    // keeps its place in the issuer's schedule with these.
    auto keep_rounds = [&](int from) {
      __syncwarp();
      if (kDq) {
        if (from < 1) named_bar_sync(bar_tile(kRoundT1Read, n), kTileThreads);
        if (from < 2) named_bar_sync(bar_tile(kRoundT2Read, n), kTileThreads);
      } else if (from < 1) {
        named_bar_sync(bar_tile(kRoundP0, n), kHalfThreads);
        named_bar_sync(bar_tile(kRoundP1, n), kTileThreads);
      }
      named_bar_sync(bar_tile(kRoundDs, n), kDsThreads<kDq>);
    };
    // dQ: the statistics of this row in the item after the current one, loaded an item ahead
    // (from L2, where the launch before dK/dV has left them: this launch has not waited for it).
    Items ahead(p, slot);
    float next_lse = 0.f, next_delta = 0.f;
    auto load_stats = [&]() {
      if (!ahead.next_busy()) return;
      const float* st = p.stats + (static_cast<long long>(ahead.head) * p.nq + ahead.tile) * (2 * kTile);
      next_lse = __ldcg(st + row);
      next_delta = __ldcg(st + kTile + row);
    };
    if (kDq) load_stats();
    const uint32_t tT1 = tBase + kColT1, tT2 = tBase + kColT2;
    int full_lo = 0, full_hi = 0;
    // One tile.  Returns -1, or the first of the tile's barrier rounds that an abort kept it
    // from.
    auto one_tile = [&](bool masked) -> int {
      const uint32_t phase = (n >> 1) & 1;
      bool ok;
      {
        const uint32_t t1 = bar(B_T1_FULL + static_cast<int>(n & 1)), st = bar(B_STAT + static_cast<int>(n & 1));
        if (kDq) {
          ok = wait_phase(t1, phase, watch);
        } else {
          // Both probes in flight together: usually both have completed.
          const uint32_t a = mbar_try_wait(t1, phase), b = mbar_try_wait(st, phase);
          ok = (a && b) || (wait_phase(t1, phase, watch) && wait_phase(st, phase, watch));
        }
      }
      if (!__all_sync(0xffffffffu, ok)) return 0;
      tc_fence_after();
      AVO_TRACE_HOOK(wg, n, 0);
      // A tile that some row of the warp does not see whole: hidden scores become -inf in
      // place, so that the code below is the same for every tile.  (Measured on B200, B4 H16
      // S4096, both passes: a test behind the exponentials or a second copy of the code cost
      // 7 to 20 %: the one splits the block that the scheduler interleaves, the other spills.)
      if (masked) {
        const int r = it.items.tile * kTile + row, c0 = it.t * kTile;
        const int lo = kDq ? 0 : r - offset - c0;
        const int hi = kDq ? (causal ? min(p.seq_kv, r + offset + 1) : p.seq_kv) - c0 : kTile;
#pragma unroll 1
        for (int c = 0; c < kTile; c += 64) {
          uint32_t s[16];
          tmem_ld16(tT1 + c, s);
          tmem_wait_ld16(s);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int col = c + wg * 16 + i;
            s[i] = col >= lo && col < hi ? s[i] : 0xff800000u;
          }
          tmem_st8(tT1 + c, s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7]);
          tmem_st8(tT1 + c + 8, s[8], s[9], s[10], s[11], s[12], s[13], s[14], s[15]);
        }
        tc_wait_st();
      }
      // P: fp32 pairs kept for dS, bf16 to TMEM (dK/dV only) a half at a time, so that dV's
      // first MMAs overlap the second half's exponentials.
      uint64_t pr[16];
      {
        uint32_t s[2][16];
        tmem_ld16(tT1, s[0]);
        tmem_ld16(tT1 + 64, s[1]);
        const uint32_t stat = sbase + kSmStat + (n & 1) * kStatBytes + wg * 64;
        const uint64_t neg2 = f2_pack(neg_lse, neg_lse);
        tmem_wait_ld16(s[0]);
        tmem_wait_ld16(s[1]);
        if (kDq) {
          // S_{n+1} may overwrite T1.
          tc_fence_before();
          __syncwarp();
          named_bar_arrive(bar_tile(kRoundT1Read, n), kTileThreads);
        }
        AVO_TRACE_HOOK(wg, n, 1);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            uint64_t la = neg2, lb = neg2;
            if (!kDq) lds_f2x2(stat + (c * 64 + e * 2) * 4, la, lb);
            pr[c * 8 + e] = exp2_pair<kEmu>(e, f2_fma(f2_pack(u2f(s[c][2 * e]), u2f(s[c][2 * e + 1])), scale2, la));
            pr[c * 8 + e + 1] =
                exp2_pair<kEmu>(e + 1, f2_fma(f2_pack(u2f(s[c][2 * e + 2]), u2f(s[c][2 * e + 3])), scale2, lb));
          }
          if (!kDq) {
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = pack_pair(pr[c * 8 + i]);
            tmem_st8(tT1 + c * 64, w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]);
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            named_bar_arrive(bar_tile(c == 0 ? kRoundP0 : kRoundP1, n), c == 0 ? kHalfThreads : kTileThreads);
          }
        }
      }
      AVO_TRACE_HOOK(wg, n, 2);
      if (!__all_sync(0xffffffffu, wait_phase(bar(B_T2_FULL + static_cast<int>(n & 1)), phase, watch))) return 1;
      tc_fence_after();
      AVO_TRACE_HOOK(wg, n, 3);
      {
        uint32_t d[2][16];
        tmem_ld16(tT2, d[0]);
        tmem_ld16(tT2 + 64, d[1]);
        tmem_wait_ld16(d[0]);
        tmem_wait_ld16(d[1]);
        if (kDq) {
          // dP_{n+1} may overwrite T2 while dS_n is computed.
          tc_fence_before();
          __syncwarp();
          named_bar_arrive(bar_tile(kRoundT2Read, n), kTileThreads);
        }
        const uint32_t stat = sbase + kSmStat + (n & 1) * kStatBytes + kTile * 4 + wg * 64;
        const uint64_t neg2 = f2_pack(neg_delta, neg_delta);
        const uint32_t tDs = kDq ? tBase - wg * 8 + kColDs : tT2;
        if (kDq && n > 0) {
          // dQ_{n-1} has read the previous dS.
          const uint32_t u = n - 1;
          if (!__all_sync(0xffffffffu,
                          wait_phase(bar(B_Y1_EMPTY + static_cast<int>(u % kY1)), (u / kY1) & 1, watch)))
            return 2;
          tc_fence_after();
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t w[8];
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            uint64_t la = neg2, lb = neg2;
            if (!kDq) lds_f2x2(stat + (c * 64 + e * 2) * 4, la, lb);
            w[e] = pack_pair(f2_mul(pr[c * 8 + e], f2_add(f2_pack(u2f(d[c][2 * e]), u2f(d[c][2 * e + 1])), la)));
            w[e + 1] = pack_pair(
                f2_mul(pr[c * 8 + e + 1], f2_add(f2_pack(u2f(d[c][2 * e + 2]), u2f(d[c][2 * e + 3])), lb)));
          }
          tmem_st8(tDs + c * (kDq ? 32 : 64), w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]);
        }
      }
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      named_bar_arrive(bar_tile(kRoundDs, n), kDsThreads<kDq>);
      AVO_TRACE_HOOK(wg, n, 4);
      return -1;
    };
    int failed = -1;
    for (; it.next(); ++n) {
      if (it.first) {
        // Every row of the warp sees all columns of the tiles from full_lo up to full_hi.
        const int r0 = it.items.tile * kTile + wq * 32;  // the warp's first row
        full_lo = 0;
        full_hi = INT_MAX;
        if (kDq) {
          full_hi = causal ? max(0, min(p.seq_kv, r0 + offset + 1)) / kTile : p.seq_kv / kTile;
          neg_lse = next_lse;
          neg_delta = next_delta;
          load_stats();
        } else if (causal) {
          full_lo = (max(0, r0 + 31 - offset) + kTile - 1) / kTile;
        }
      }
      failed = one_tile(it.t < full_lo || it.t >= full_hi);
      if (failed >= 0) break;
    }
    if (failed >= 0) {
      keep_rounds(failed);
      for (++n; it.next(); ++n) keep_rounds(0);
    }
  } else if (warp < kProducerWarp) {
    if constexpr (kBwdRegsEpi < kBwdRegsLaunch) regs_decrease<kBwdRegsEpi>();
    // ------------------------------------------------------------ epilogue
    const int row = threadIdx.x & 127;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const int rows = kDq ? p.seq_q : p.seq_kv;
    bool ok = true;
    uint32_t done = 0;   // items with tiles so far
    // dQ: this thread's row of Q of the next item with tiles, its first half loaded an item
    // ahead, the second when it is stored.
    Items ahead(p, slot);
    uint32_t xq[32];
    bool have_x = false;
    auto load_half = [&](int half) {
      const int r = ahead.tile * kTile + row;
      const bool valid = r < rows;
      const uint4* src =
          static_cast<const uint4*>(p.x1) + (static_cast<long long>(ahead.head) * rows + (valid ? r : 0)) * 16 + half * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint4 v = valid ? __ldg(src + i) : make_uint4(0u, 0u, 0u, 0u);
        xq[4 * i] = v.x;
        xq[4 * i + 1] = v.y;
        xq[4 * i + 2] = v.z;
        xq[4 * i + 3] = v.w;
      }
    };
    auto load_x = [&]() {
      have_x = ahead.next_busy();
      if (have_x) load_half(0);
    };
    uint32_t x_signals = 0, acc_signals = 0;
    auto store_x = [&]() {
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        if (half == 1) load_half(1);
        const uint32_t t = tmem + lane_off + kColX1 + half * 32;
#pragma unroll
        for (int i = 0; i < 32; i += 8)
          tmem_st8(t + i, xq[i], xq[i + 1], xq[i + 2], xq[i + 3], xq[i + 4], xq[i + 5], xq[i + 6], xq[i + 7]);
      }
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      named_bar_arrive(bar_x1(x_signals++), kEpiThreads);
    };
    if (kDq) {
      load_x();
      if (have_x) store_x();
    }
    Items it(p, slot);
    while (ok && it.next()) {
      if (kDq && it.n > 0) {
        load_x();
        if (have_x) {
          // Q may be replaced once this item's last S is done with it.
          ok = wait_item(bar(B_X1_DONE), done & 1, it.n, watch, lane);
          if (!ok) break;
          tc_fence_after();
          store_x();
        }
      }
      const int r = it.tile * kTile + row;
      const bool write = r < rows;
      const long long at = (static_cast<long long>(it.head) * rows + r) * kHeadDim;
      const long long part_at =
          ((static_cast<long long>(it.piece) * (kDq ? p.q_heads : p.kv_heads) + it.head) * rows + r) * kHeadDim;
      // dK/dV: dV (accumulator 2, complete first), then dK; dQ: accumulator 1 only.
#pragma unroll 1
      for (int a = kDq ? 1 : 2; a >= 1; --a) {
        __nv_bfloat16* const dst = static_cast<__nv_bfloat16*>(a == 1 ? p.g1 : p.g2) + at;
        float* const part = (a == 1 ? p.part1 : p.part2) + part_at;
        const float f = a == 1 ? p.scale : 1.f;
        const uint32_t acc = tmem + lane_off + (a == 1 ? kColAcc1 : kColAcc2);
        if (it.n > 0) {
          ok = wait_item(bar(a == 1 ? B_ACC1 : B_ACC2), done & 1, it.n, watch, lane);
          if (!ok) break;
          tc_fence_after();
        }
        // The next 16 columns are on their way while these are stored.
        uint32_t o[2][16];
        if (it.n > 0) {
          tmem_ld16(acc, o[0]);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) o[0][e] = o[1][e] = 0u;
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          uint32_t* const x = o[c & 1];
          if (it.n > 0) {
            tmem_wait_ld16(o[c & 1]);
            if (c < 7) {
              tmem_ld16(acc + (c + 1) * 16, o[(c + 1) & 1]);
            } else {
              // Read out: the next item may overwrite it.
              tc_fence_before();
              __syncwarp();
              named_bar_arrive(a == 1 ? bar_acc1(done) : bar_acc2(done), kEpiThreads);
              ++acc_signals;
            }
          }
          if (kOrder == kAny && write && p.split > 1) {
#pragma unroll
            for (int e = 0; e < 16; e += 8)
              st_global_v8(part + c * 16 + e, x[e], x[e + 1], x[e + 2], x[e + 3], x[e + 4], x[e + 5], x[e + 6], x[e + 7]);
          } else if (write) {
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = pack_bf16x2(u2f(x[2 * e]) * f, u2f(x[2 * e + 1]) * f);
            st_global_v8(dst + c * 16, w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]);
          }
        }
      }
      if (it.n > 0) ++done;
    }
    if (!ok) {
      // After an abort: the signals not given yet, as blocking syncs in the issuer's order.
      __syncwarp();
      uint32_t x_seen = 0, acc_seen = 0, item = 0;
      auto x_round = [&]() {
        if (x_seen >= x_signals) named_bar_sync(bar_x1(x_seen), kEpiThreads);
        ++x_seen;
      };
      auto acc_round = [&](uint32_t i) {
        if (!kDq && acc_seen++ >= acc_signals) named_bar_sync(bar_acc2(i), kEpiThreads);
        if (acc_seen++ >= acc_signals) named_bar_sync(bar_acc1(i), kEpiThreads);
      };
      Items all(p, slot), after(p, slot);
      bool more = after.next_busy();
      if (kDq && more) x_round();
      for (; all.next_busy(); ++item) {
        more = after.next_busy();
        if (kDq && more && all.n == 1) x_round();
        if (item > 0) acc_round(item - 1);
        if (kDq && more && all.n > 1) x_round();
        if (!more) acc_round(item);
      }
    }
  } else if (warp == kProducerWarp) {
    regs_decrease<kBwdRegsOther>();
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      const uint64_t pol_x = policy_evict_first();
      const uint64_t pol_y = policy_evict_last();
      auto load = [&](int off, const CUtensorMap* tm, int b, int r0, int head, uint64_t pol) {
        mbar_arrive_expect_tx(bar(b), kTileBytes);
        tma_load_3d(sbase + off, tm, bar(b), 0, r0, head, pol);
        tma_load_3d(sbase + off + kHalfBytes, tm, bar(b), 64, r0, head, pol);
      };
      // A buffer may be loaded again once its last user is done.  That it is done also means
      // that its previous copy has landed, unless the CTA aborted before: then the MMAs no
      // longer waited for data.  The flag is set before any such MMA is issued, so it is seen
      // here after its commit: at most one copy per buffer is ever in flight.  (No more than
      // these two reads of shared memory per load: each takes 100 to 300 cycles while the MMAs
      // read their operands.)
      auto reuse_after = [&](int done, uint32_t parity) {
        return wait_phase(bar(done), parity, watch) && !*abort_flag;
      };
      // ... done as tile u's T1 or T2 commit implies.
      auto reuse = [&](int commit, int u) { return reuse_after(commit + (u & 1), (u >> 1) & 1); };
      int n = 0, n2 = 0, nx1 = 0, nx2 = 0, nst = 0, skipped = -1;
      // The stationary tiles of the next item, and its first streamed ones, are brought to L2
      // while this item runs, once its own first loads are on their way: their loads start only
      // when its last tiles are done with the buffers.
      Items ahead(p, slot);
      ahead.next_busy();
      auto prefetch = [&](const CUtensorMap* tm, int r0, int head) {
        tma_prefetch_3d(tm, 0, r0, head);
        tma_prefetch_3d(tm, 64, r0, head);
      };
      Tiles it(p, slot);
      while (it.next()) {
        const int s1 = n % kY1, s2 = n % kY2;
        // Y1's last user is its tile's last MMA: dQ, or dK, which precedes the next tile's T2.
        if (n >= kY1 && !(kDq ? reuse_after(B_Y1_EMPTY + s1, (n / kY1 - 1) & 1) : reuse(B_T2_FULL, n - 2))) break;
        if (n == p.test_skip_load) skipped = n;  // test hook: this copy never arrives
        if (n != skipped) load(Sm::kY1At + s1 * kTileBytes, &tm_y1, B_Y1_FULL + s1, it.t * kTile, it.y_head, pol_y);
        ++n;
        const int last = n - 2;  // the previous tile
        if (!kDq && it.first) {
          // X1 was read last by the previous tile's T1, X2 by its T2.
          if (nx1 > 0 && !reuse(B_T1_FULL, last)) break;
          load(Sm::kX1, &tm_x1, B_X1_FULL, it.items.tile * kTile, it.items.head, pol_x);
          ++nx1;
        }
        // Y2's last user is dV, or T2 itself (dQ).
        if (n2 >= kY2 && !(kDq ? reuse(B_T2_FULL, last - 1) : reuse_after(B_Y2_EMPTY + s2, (n2 / kY2 - 1) & 1))) break;
        load(Sm::kY2At + s2 * kTileBytes, &tm_y2, B_Y2_FULL + s2, it.t * kTile, it.y_head, pol_y);
        ++n2;
        if (it.first) {
          if (nx2 > 0 && !reuse(B_T2_FULL, last)) break;
          load(Sm::kX2, &tm_x2, B_X2_FULL, it.items.tile * kTile, it.items.head, pol_x);
          ++nx2;
        }
        if (!kDq) {
          // The slot's last readers published dS of tile nst - 2 before that tile's dK, which
          // precedes T2 of tile nst - 1.
          const int slot = nst & 1;
          if (nst >= 2 && !reuse(B_T2_FULL, nst - 1)) break;
          const float* src = p.stats + (static_cast<long long>(it.y_head) * p.nq + it.t) * (2 * kTile);
          mbar_arrive_expect_tx(bar(B_STAT + slot), kStatBytes);
          bulk_load(sbase + kSmStat + slot * kStatBytes, src, kStatBytes, bar(B_STAT + slot));
          ++nst;
        }
        if (it.first && ahead.next_busy()) {
          const int y_head = kDq ? ahead.head / p.group : ahead.head * p.group;
          if (!kDq) prefetch(&tm_x1, ahead.tile * kTile, ahead.head);
          prefetch(&tm_x2, ahead.tile * kTile, ahead.head);
          prefetch(&tm_y1, (ahead.t0 + (kDq ? ahead.skip : 0)) * kTile, y_head);
          prefetch(&tm_y2, (ahead.t0 + (kDq ? ahead.skip : 0)) * kTile, y_head);
        }
      }
      if (*abort_flag) {
        // Copies already issued still land in shared memory: wait for them.
        for (int u = max(0, n - kY1); u < n; ++u)
          if (u != skipped) drain_phase(bar(B_Y1_FULL + u % kY1), (u / kY1) & 1, watch);
        for (int u = max(0, n2 - kY2); u < n2; ++u) drain_phase(bar(B_Y2_FULL + u % kY2), (u / kY2) & 1, watch);
        for (int u = max(0, nst - 2); u < nst; ++u) drain_phase(bar(B_STAT + (u & 1)), (u >> 1) & 1, watch);
        if (nx1 > 0) drain_phase(bar(B_X1_FULL), (nx1 - 1) & 1, watch);
        if (nx2 > 0) drain_phase(bar(B_X2_FULL), (nx2 - 1) & 1, watch);
      }
    }
    __syncwarp();
  } else if (warp == kIssuerWarp) {
    regs_decrease<kBwdRegsOther>();
    // ------------------------------------------------------------ MMA issuer
    // The issuing lane is chosen by elect.sync: with `lane == 0` issuing was the limit
    // (measured on B200, B1 H16 S4096: 3324 and 2731 cycles per tile pair of the two passes,
    // 2814 and 2104 with elect.sync).
    const bool leader = elect_one();
    const uint32_t tT1 = tmem + kColT1, tT2 = tmem + kColT2, tA1 = tmem + kColAcc1, tA2 = tmem + kColAcc2;
    const uint32_t tDs = tmem + kColDs, tX1 = tmem + kColX1;
    const uint32_t x1 = smem_desc_lo(sbase + Sm::kX1, 16), x2 = smem_desc_lo(sbase + Sm::kX2, 16);
    // Streamed tiles as the N x K operand of T1 and T2, and as the K x N operand of the
    // accumulating MMAs.
    const uint32_t y1 = smem_desc_lo(sbase + Sm::kY1At, 16), y1t = smem_desc_lo(sbase + Sm::kY1At, kHalfBytes);
    const uint32_t y2 = smem_desc_lo(sbase + Sm::kY2At, 16), y2t = smem_desc_lo(sbase + Sm::kY2At, kHalfBytes);
    constexpr uint32_t kSlot = kTileBytes >> 4;
    auto sync_on = [&](uint32_t id, uint32_t threads) {
      __syncwarp();
      named_bar_sync(id, threads);
      tc_fence_after();
    };
    Tiles it(p, slot);
    uint32_t items = 0;
    auto issue_t1 = [&](int slot, int parity) {
      if constexpr (kDq)
        issue_xy_tmem(tT1, tX1, y1 + slot * kSlot);
      else
        issue_xy(tT1, x1, y1 + slot * kSlot);
      mma_commit(bar(B_T1_FULL + parity));
      if (kDq && it.last) mma_commit(bar(B_X1_DONE));
    };
    auto issue_t2 = [&](int parity) {  // the parity is also the Y2 slot
      issue_xy(tT2, x2, y2 + parity * kSlot);
      mma_commit(bar(B_T2_FULL + parity));
    };
    bool have = it.next();
    if (have) {
      sync_on(kBarLoaded, 64);
      if (kDq) sync_on(bar_x1(0), kEpiThreads);
      if (leader) issue_t1(0, 0);
      sync_on(kBarLoaded, 64);
      if (leader) issue_t2(0);
    }
    int s1 = 0, par = 0;  // Y1 slot of the current tile; its parity
    while (have) {
      const bool first = it.first, last = it.last;
      have = it.next();  // now: the tile after the current one
      const int n1 = s1 == kY1 - 1 ? 0 : s1 + 1, other = par ^ 1;
      if constexpr (!kDq) {
        if (first && items > 0) sync_on(bar_acc2(items - 1), kEpiThreads);
        sync_on(bar_tile(kRoundP0, par), kHalfThreads);
        if (leader) issue_acc_half<false>(tA2, tT1, y2t + par * kSlot, 0, first ? 0u : 1u);
        sync_on(bar_tile(kRoundP1, par), kTileThreads);
        if (leader) {
          issue_acc_half<false>(tA2, tT1, y2t + par * kSlot, 1, 1u);
          mma_commit(bar(B_Y2_EMPTY + par));
          if (last) mma_commit(bar(B_ACC2));
          if (have) issue_t1(n1, other);
        }
        if (first && items > 0) sync_on(bar_acc1(items - 1), kEpiThreads);
        sync_on(bar_tile(kRoundDs, par), kTileThreads);
        if (leader) {
          issue_acc<false>(tA1, tT2, y1t + s1 * kSlot, first ? 0u : 1u);
          if (last) mma_commit(bar(B_ACC1));
          if (have) issue_t2(other);
        }
      } else {
        sync_on(bar_tile(kRoundT1Read, par), kTileThreads);
        if (have && it.first) sync_on(bar_x1(items + (first ? 1 : 0)), kEpiThreads);
        if (leader && have) issue_t1(n1, other);
        sync_on(bar_tile(kRoundT2Read, par), kTileThreads);
        if (leader && have) issue_t2(other);
        if (first && items > 0) sync_on(bar_acc1(items - 1), kEpiThreads);
        sync_on(bar_tile(kRoundDs, par), kHalfThreads);
        if (leader) {
          issue_acc<true>(tA1, tDs, y1t + s1 * kSlot, first ? 0u : 1u);
          mma_commit(bar(B_Y1_EMPTY + s1));
          if (last) mma_commit(bar(B_ACC1));
        }
      }
      if (first) ++items;
      s1 = n1;
      par = other;
    }
    if (items > 0) {
      if (!kDq) sync_on(bar_acc2(items - 1), kEpiThreads);
      sync_on(bar_acc1(items - 1), kEpiThreads);
    }
    __syncwarp();
    if (leader && items > 0) {
      // Every MMA completes before TMEM and shared memory are released.
      mma_commit(bar(B_DRAINED));
      drain_phase(bar(B_DRAINED), 0, watch);
    }
    __syncwarp();
  } else if (warp == kWaiterWarp) {
    regs_decrease<kBwdRegsOther>();
    // ------------------------------------------------------------ waiter
    // The loads' mbarrier waits in the issuer's order (X1 and Y1 of a tile for T1, X2 and Y2
    // for T2); then its rounds on the barriers whose release lets the issuer use them.  After
    // an abort the waits return at once and only the rounds are kept.
    int n1 = 0, n2 = 0, x1 = 0, x2 = 0;
    Tiles a(p, slot), c(p, slot);  // tiles whose T1 / T2 operands are next
    auto t1_loaded = [&]() {
      if (!a.next()) return;
      if (lane == 0) {
        if (!kDq && a.first) wait_phase(bar(B_X1_FULL), x1 & 1, watch);
        wait_phase(bar(B_Y1_FULL + n1 % kY1), (n1 / kY1) & 1, watch);
      }
      if (a.first) ++x1;
      ++n1;
    };
    auto t2_loaded = [&]() {
      if (!c.next()) return;
      if (lane == 0) {
        if (c.first) wait_phase(bar(B_X2_FULL), x2 & 1, watch);
        wait_phase(bar(B_Y2_FULL + n2 % kY2), (n2 / kY2) & 1, watch);
      }
      if (c.first) ++x2;
      ++n2;
    };
    auto round = [&](uint32_t id, uint32_t threads) {
      __syncwarp();
      named_bar_sync(id, threads);
    };
    Tiles it(p, slot);
    bool have = it.next();
    if (have) {
      t1_loaded();
      round(kBarLoaded, 64);
      t2_loaded();
      round(kBarLoaded, 64);
    }
    for (uint32_t n = 0; have; have = it.next(), ++n) {
      t1_loaded();
      round(bar_tile(kDq ? kRoundT1Read : kRoundP1, n), kTileThreads);
      t2_loaded();
      round(bar_tile(kDq ? kRoundT2Read : kRoundDs, n), kTileThreads);
    }
  } else {
    regs_decrease<kBwdRegsOther>();  // warp 23 completes the warpgroup
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kIssuerWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
  // The dQ launch is complete only when the dK/dV launch is (see above).  One CTA waits for
  // that; the others make room.
  if (kDq && blockIdx.x == gridDim.x - 1) grid_dependency_wait();
}

// The sums of split units: out = bf16(factor * (part[0] + part[1] + ...)), in this order, for
// up to three gradients (dK, dV, dQ; count 0: not split).  8 values per thread.
struct JoinParams {
  const float* part[3];
  __nv_bfloat16* out[3];
  float factor[3];
  uint32_t pieces[3];
  long long count[3];    // groups of 8 values
};

__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ JoinParams p) {
  grid_dependency_wait();
  long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  int g = 0;
  while (g < 3 && i >= p.count[g]) i -= p.count[g++];
  if (g == 3) return;
  const float4* src = reinterpret_cast<const float4*>(p.part[g]) + 2 * i;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
#pragma unroll 4
  for (uint32_t k = 0; k < p.pieces[g]; ++k) {
    const float4 c = __ldcg(src), d = __ldcg(src + 1);
    src += 2 * p.count[g];
    a.x += c.x; a.y += c.y; a.z += c.z; a.w += c.w;
    b.x += d.x; b.y += d.y; b.z += d.z; b.w += d.w;
  }
  const float f = p.factor[g];
  reinterpret_cast<uint4*>(p.out[g])[i] = make_uint4(pack_bf16x2(a.x * f, a.y * f), pack_bf16x2(a.z * f, a.w * f),
                                                     pack_bf16x2(b.x * f, b.y * f), pack_bf16x2(b.z * f, b.w * f));
}

// -LSE*log2(e) and -delta of every query row, padded to whole tiles: [heads][nq][2][128].
// 16 lanes per row, 16 bytes of O and dO each, four rows at a time (measured on B200, B2 H16
// S4001 back to back, the whole gradient: one row at a time 422.6 us, four 420).  Rows past seq_q
// and rows that saw no key (LSE = -inf) get -inf, so their probabilities are exactly 0.
constexpr int kStatRows = 4;                     // rows per half-warp, all in flight at once
constexpr int kStatBlockRows = 16 * kStatRows;   // rows per block

__global__ void __launch_bounds__(256)
    stats_kernel(const uint4* __restrict__ dout, const uint4* __restrict__ out, const float* __restrict__ lse,
                 float* __restrict__ stats, int seq_q, int nq, uint32_t* claims) {
  grid_dependency_wait();
  grid_launch_dependents();
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < 2 * kMaxClaims; i += blockDim.x) claims[i] = 0u;
  // Blocks cover the padded rows exactly (128 of every tile), each within one tile.
  const int l = threadIdx.x & 15;
  const long long tile = blockIdx.x / (kTile / kStatBlockRows);
  const int r0 = static_cast<int>(blockIdx.x % (kTile / kStatBlockRows)) * kStatBlockRows +
                 static_cast<int>(threadIdx.x >> 4) * kStatRows;
  const long long head = tile / nq;
  const int row0 = static_cast<int>(tile % nq) * kTile + r0;
  uint4 a[kStatRows], b[kStatRows];
#pragma unroll
  for (int k = 0; k < kStatRows; ++k) {
    const bool valid = row0 + k < seq_q;
    const long long at = (head * seq_q + (valid ? row0 + k : 0)) * 16 + l;
    a[k] = valid ? dout[at] : make_uint4(0u, 0u, 0u, 0u);
    b[k] = valid ? out[at] : make_uint4(0u, 0u, 0u, 0u);
  }
  float mine = 0.f;  // of row l, in the first lanes
#pragma unroll
  for (int k = 0; k < kStatRows; ++k) {
    const uint32_t wa[4] = {a[k].x, a[k].y, a[k].z, a[k].w}, wb[4] = {b[k].x, b[k].y, b[k].z, b[k].w};
    float acc = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      acc = fmaf(u2f(wa[i] << 16), u2f(wb[i] << 16), acc);
      acc = fmaf(u2f(wa[i] & 0xffff0000u), u2f(wb[i] & 0xffff0000u), acc);
    }
#pragma unroll
    for (int m = 8; m > 0; m >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, m);
    if (l == k) mine = acc;
  }
  if (l < kStatRows) {
    float neg = -CUDART_INF_F;
    if (row0 + l < seq_q) {
      const float v = lse[head * seq_q + row0 + l];
      neg = v == -CUDART_INF_F ? v : -v * 1.4426950408889634f;
    }
    float* dst = stats + tile * (2 * kTile) + r0 + l;
    dst[0] = neg;
    dst[kTile] = -mine;
  }
}

}  // namespace bwd
}  // namespace avo_b200
