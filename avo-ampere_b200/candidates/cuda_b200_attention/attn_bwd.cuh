// Gradient of attention for sm_100a (B200), head_dim 128, bf16 in and out.
//
// With S = scale * Q K^T, P = exp(S - LSE) (0 where the mask hides the key), dP = dO V^T and
// delta_i = sum_d dO_id O_id:
//     dS = P * (dP - delta),  dQ = scale * dS K,  dK = scale * dS^T Q,  dV = P^T dO,
// dK and dV summed over the query heads that share a key/value head.  The probabilities are
// recomputed from Q, K and the LSE the forward saved.
//
// Three launches.  stats_kernel writes -LSE*log2(e) and -delta per query row.  Then one
// kernel template runs twice over 128 x 128 tiles, each time with one side of the tile
// stationary in shared memory and the other streamed:
//
//             rows (M)   stationary X1, X2   streamed Y1, Y2   accumulators in TMEM
//   dK/dV     keys       K, V                Q, dO             dK += dS^T Q, dV += P^T dO
//   dQ        queries    Q, dO               K, V              dQ += dS K
//
//   T1 = X1 Y1^T (S or S^T), T2 = X2 Y2^T (dP or dP^T); the softmax warps turn them into P
//   and dS, bf16, in place in TMEM, where they are the A operand of the accumulating MMAs.
//
// Two passes recompute S and dP: 7 products per tile pair instead of the 5 that one pass
// needs.  In exchange dQ is not accumulated across CTAs: no atomics (the result does not
// depend on the order in which CTAs run), no fp32 dQ in memory, and neither P nor dS ever
// leaves TMEM.  With one 128 x 128 tile in flight per pass the tensor pipe is what bounds
// both passes: per tile it needs 2048 (dK/dV) and 1536 (dQ) cycles, and the 256 softmax
// threads' work on it overlaps, phase against phase:
//
//   dK/dV:  tensor   | dV_n  S_{n+1} | dK_n  dP_{n+1} | dV_{n+1} ...
//           softmax  | dS_n from dP_n | P_{n+1} from S_{n+1} | ...
//   dQ:     tensor   | dP_{n+1}  dQ_n  S_{n+2} | ...           (S double buffered)
//           softmax  | P_{n+1} from S_{n+1}, dS_{n+1} from dP_{n+1} | ...
//
// Sums are fp32 in TMEM; P and dS are rounded once to bf16 (the type of the tensor cores'
// operands: half a step, 2^-9 of each value), the gradients once at the end.
//
// Roles (512 threads): warps 0-7 softmax (two warpgroups, 64 of a tile's 128 columns each),
// warps 8-11 the epilogue (an item's accumulators to memory while the next item's first
// tiles run), warp 12 TMA producer, warp 13 MMA issuer, warp 14 waiter: the issuer waits on
// hardware named barriers only, because a shared-memory read by the issuing thread drains
// its queued MMAs first.  Every wait is bounded by the watchdog, and after an abort every
// role still takes its fixed number of barrier rounds, so no CTA is left waiting.
#pragma once

#include <cuda_bf16.h>

#include "attn_fwd.cuh"

namespace avo_b200 {
namespace bwd {

constexpr int kTile = 128;
constexpr int kSoftmaxThreads = 256;
constexpr int kEpiWarp = 8;
constexpr int kProducerWarp = 12;
constexpr int kIssuerWarp = 13;
constexpr int kWaiterWarp = 14;
constexpr int kBwdThreads = 512;
// Launched at 128 registers per thread (512 x 128 = 65536); 256 x 168 + 128 x 96 + 128 x 72
// = 64512 after the split.
constexpr uint32_t kBwdRegsLaunch = 128;
constexpr uint32_t kBwdRegsSoftmax = 168;
constexpr uint32_t kBwdRegsEpi = 96;
constexpr uint32_t kBwdRegsOther = 72;
static_assert(256 * kBwdRegsSoftmax + 128 * kBwdRegsEpi + 128 * kBwdRegsOther <= kBwdThreads * kBwdRegsLaunch,
              "register split");

// Named barriers: 3 waiter -> issuer, 4 P in TMEM, 5 dS in TMEM (the 8 softmax warps arrive,
// the issuer syncs), 6 / 7 accumulator 1 / 2 read out (the epilogue warps arrive).
constexpr uint32_t kBarLoaded = 3;
constexpr uint32_t kBarP = 4;
constexpr uint32_t kBarDs = 5;
constexpr uint32_t kBarAcc1 = 6;
constexpr uint32_t kBarAcc2 = 7;

// Y1 (used by T1 and by the last MMA of its tile) has three slots and Y2 two: with two Y1
// slots a tile's load could only start 1024 tensor cycles before its use, about the latency
// of a 32 KB load.
constexpr int kY1 = 3;
constexpr int kY2 = 2;
constexpr int kSmX1 = 0;
constexpr int kSmX2 = kTileBytes;
constexpr int kSmY1 = 2 * kTileBytes;
constexpr int kSmY2 = kSmY1 + kY1 * kTileBytes;
constexpr int kSmStat = kSmY2 + kY2 * kTileBytes;  // two slots of [-LSE*log2 e | -delta], 128 floats each
constexpr int kStatBytes = 2 * kTile * 4;
constexpr int kSmBars = kSmStat + 2 * kStatBytes;
enum : int {
  B_X1_FULL = 0,
  B_X2_FULL,
  B_X1_EMPTY,
  B_X2_EMPTY,
  B_Y1_FULL,
  B_Y1_EMPTY = B_Y1_FULL + kY1,
  B_Y2_FULL = B_Y1_EMPTY + kY1,
  B_Y2_EMPTY = B_Y2_FULL + kY2,
  B_T1_FULL = B_Y2_EMPTY + kY2,  // two: dQ's T1 is double buffered
  B_T2_FULL = B_T1_FULL + 2,
  B_ACC1,
  B_ACC2,
  B_STAT,
  B_DRAINED = B_STAT + 2,
  B_COUNT
};
constexpr int kSmTmem = kSmBars + B_COUNT * 8;
constexpr int kSmAbort = kSmTmem + 4;
constexpr int kBwdSmemBytes = (kSmAbort + 4 + 15) / 16 * 16;
static_assert(kBwdSmemBytes <= 227 * 1024, "shared memory budget");

// TMEM columns: T1 | T2 | accumulator 1 | accumulator 2 (dK/dV) or T1's second buffer (dQ).
constexpr uint32_t kColT1 = 0, kColT2 = 128, kColAcc1 = 256, kColAcc2 = 384;

struct BwdParams {
  const float* stats;  // [num_q_heads][nq][2][128]: -LSE*log2(e), -delta
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
  int test_skip_load;
};

// One CTA's items in order: (stationary tile of one head), waves over the grid in alternating
// directions, causal items longest first.
template <bool kDq>
struct Items {
  const BwdParams& p;
  int r = 0;
  int head, tile;  // stationary head and tile
  int t0, n;       // first streamed tile, tiles in all (dK/dV: over the whole group of heads)
  __device__ explicit Items(const BwdParams& params) : p(params) {}
  __device__ bool next() {
    const int heads = kDq ? p.q_heads : p.kv_heads;
    const int tiles = kDq ? p.nq : p.nkv;
    const int count = heads * tiles;
    const int grid = static_cast<int>(gridDim.x), cta = static_cast<int>(blockIdx.x);
    while (true) {
      const long long base = static_cast<long long>(r) * grid;
      if (base >= count) return false;
      const long long w64 = base + ((r & 1) ? grid - 1 - cta : cta);
      ++r;
      if (w64 >= count) continue;
      const int w = static_cast<int>(w64);
      if (p.causal) {
        head = w % heads;
        tile = kDq ? tiles - 1 - w / heads : w / heads;
      } else {
        head = w / tiles;
        tile = w % tiles;
      }
      if (kDq) {
        t0 = 0;
        n = p.nkv;
        if (p.causal) {
          const int q_end = min(tile * kTile + kTile, p.seq_q);
          const int last = q_end - 1 + p.offset;  // last key any row sees
          n = last < 0 ? 0 : min(p.nkv, last / kTile + 1);
        }
      } else {
        t0 = 0;
        if (p.causal) t0 = min(max(0, tile * kTile - p.offset) / kTile, p.nq);
        // A key tile past the last query's reach: max(0, k0 - offset) >= seq_q.
        if (p.causal && tile * kTile - p.offset >= p.seq_q) t0 = p.nq;
        n = (p.nq - t0) * p.group;
      }
      return true;
    }
  }
};

// The tiles of a CTA's items as one sequence (items without tiles are skipped).
template <bool kDq>
struct Tiles {
  Items<kDq> items;
  int left = 0;   // tiles of the item still to come
  int t, y_head;  // current streamed tile and its head
  bool first, last;
  __device__ explicit Tiles(const BwdParams& params) : items(params) {}
  __device__ bool next() {
    first = false;
    if (left == 0) {
      do {
        if (!items.next()) return false;
      } while (items.n == 0);
      left = items.n;
      first = true;
      t = items.t0;
      y_head = kDq ? items.head / items.p.group : items.head * items.p.group;
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

// acc (+)= A Y over the 128 streamed rows: A (P or dS, bf16) from TMEM, where each softmax
// warpgroup has put its 64 columns' values at the start of its own half of the tile; Y from
// shared memory as an MN-major operand.
__device__ __forceinline__ void issue_acc(uint32_t d_tmem, uint32_t a_tmem, uint32_t y_lo, uint32_t accumulate) {
  constexpr uint32_t idesc = idesc_bf16_f32(kTile, kHeadDim, 0, 1);
#pragma unroll
  for (int kk = 0; kk < 8; ++kk)
    mma_ts_lo(d_tmem, a_tmem + (kk >> 2) * 64 + (kk & 3) * 8, y_lo + ((kk * 16 * 128) >> 4), kDescHiSw128, idesc,
              accumulate | (kk > 0 ? 1u : 0u));
}

// 2^x for pair number `i` of a chunk: kEmu of every 8 pairs on the FMA pipe (results below
// 2^-125 become 0), the others on the MUFU unit.
template <int kEmu>
__device__ __forceinline__ uint64_t exp2_pair(int i, uint64_t x2) {
  float x0, x1, p0, p1;
  f2_unpack(x2, x0, x1);
  if ((i & 7) < kEmu) {
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

// 16 packed words to 16 TMEM columns.
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&w)[16]) {
  tmem_st8(taddr, w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]);
  tmem_st8(taddr + 8, w[8], w[9], w[10], w[11], w[12], w[13], w[14], w[15]);
}

template <bool kDq>
__global__ void __launch_bounds__(kBwdThreads, 1)
    attn_bwd_kernel(const __grid_constant__ CUtensorMap tm_x1, const __grid_constant__ CUtensorMap tm_x2,
                    const __grid_constant__ CUtensorMap tm_y1, const __grid_constant__ CUtensorMap tm_y2,
                    const __grid_constant__ BwdParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_addr(smem);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  auto bar = [&](int idx) -> uint32_t { return sbase + kSmBars + idx * 8; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kSmAbort);
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
  // launch have passed this wait: it runs on the multiprocessors that launch leaves free
  // and waits for it at its own end.
  if (!kDq) {
    grid_dependency_wait();
    grid_launch_dependents();
  }

  if (warp < kEpiWarp) {
    regs_increase<kBwdRegsSoftmax>();
    // ------------------------------------------------------------ softmax
    const int wg = warp >> 2;
    const int wq = warp & 3;
    const int row = threadIdx.x & 127;
    const uint32_t tBase = tmem + (static_cast<uint32_t>(wq * 32) << 16) + wg * 64;
    const uint64_t scale2 = f2_pack(p.scale_log2, p.scale_log2);
    bool ok = true;
    uint32_t n = 0;
    float neg_lse = 0.f, neg_delta = 0.f;
    Tiles<kDq> it(p);
    while (it.next()) {
      if (!ok) {
        // After an abort: keep this warp's place in the issuer's barrier rounds.
        __syncwarp();
        if (!kDq) named_bar_sync(kBarP, kSoftmaxThreads + 32);
        named_bar_sync(kBarDs, kSoftmaxThreads + 32);
        continue;
      }
      const uint32_t tT1 = tBase + ((kDq && (n & 1)) ? kColAcc2 : kColT1);
      const uint32_t tT2 = tBase + kColT2;
      // Columns [lo, hi) of this tile are visible to this row; mask_tile: some row of the
      // warp sees fewer than this warpgroup's 64.
      int lo = 0, hi = kTile;
      bool mask_tile;
      if (kDq) {
        const int q = it.items.tile * kTile + row;
        const int key0 = it.t * kTile;
        hi = p.seq_kv - key0;
        int hi_warp = hi;
        if (p.causal) {
          hi = min(hi, q + p.offset - key0 + 1);
          hi_warp = min(hi_warp, q - lane + p.offset - key0 + 1);
        }
        mask_tile = hi_warp < wg * 64 + 64;
        if (it.first) {
          const float* st = p.stats + (static_cast<long long>(it.items.head) * p.nq + it.items.tile) * (2 * kTile);
          neg_lse = __ldg(st + row);
          neg_delta = __ldg(st + kTile + row);
        }
      } else {
        const int key = it.items.tile * kTile + row;
        lo = p.causal ? key - p.offset - it.t * kTile : 0;
        mask_tile = p.causal && (key - lane + 31 - p.offset - it.t * kTile) > wg * 64;
      }
      const int t1_bar = kDq ? B_T1_FULL + static_cast<int>(n & 1) : B_T1_FULL;
      ok = wait_phase(bar(t1_bar), kDq ? (n >> 1) & 1 : n & 1, watch);
      if (!kDq) ok = ok && wait_phase(bar(B_STAT + static_cast<int>(n & 1)), (n >> 1) & 1, watch);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {
        if (!kDq) named_bar_sync(kBarP, kSoftmaxThreads + 32);
        named_bar_sync(kBarDs, kSoftmaxThreads + 32);
        ++n;
        continue;
      }
      tc_fence_after();
      // P for this warpgroup's 64 columns: fp32 pairs kept for dS, bf16 to TMEM (dK/dV only).
      uint64_t pr[32];
      {
        uint32_t s[2][32];
        tmem_ld32(tT1, s[0]);
        tmem_ld32(tT1 + 32, s[1]);
        tmem_wait_ld(s[0]);
        tmem_wait_ld(s[1]);
        const uint32_t stat = sbase + kSmStat + (n & 1) * kStatBytes + wg * 256;
        const uint64_t neg2 = f2_pack(neg_lse, neg_lse);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            uint64_t la = neg2, lb = neg2;
            if (!kDq) lds_f2x2(stat + (c * 32 + e * 2) * 4, la, lb);
            pr[c * 16 + e] =
                exp2_pair<2>(e, f2_fma(f2_pack(u2f(s[c][2 * e]), u2f(s[c][2 * e + 1])), scale2, la));
            pr[c * 16 + e + 1] =
                exp2_pair<2>(e + 1, f2_fma(f2_pack(u2f(s[c][2 * e + 2]), u2f(s[c][2 * e + 3])), scale2, lb));
          }
        }
      }
      if (mask_tile) {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          float a, b;
          f2_unpack(pr[i], a, b);
          const int col = wg * 64 + 2 * i;
          a = (col >= lo && col < hi) ? a : 0.f;
          b = (col + 1 >= lo && col + 1 < hi) ? b : 0.f;
          pr[i] = f2_pack(a, b);
        }
      }
      if (!kDq) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) w[i] = pack_pair(pr[c * 16 + i]);
          tmem_st16(tT1 + c * 16, w);
        }
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        named_bar_arrive(kBarP, kSoftmaxThreads + 32);
      }
      ok = __all_sync(0xffffffffu, wait_phase(bar(B_T2_FULL), n & 1, watch));
      if (!ok) {
        named_bar_sync(kBarDs, kSoftmaxThreads + 32);
        ++n;
        continue;
      }
      tc_fence_after();
      {
        uint32_t d[2][32];
        tmem_ld32(tT2, d[0]);
        tmem_ld32(tT2 + 32, d[1]);
        tmem_wait_ld(d[0]);
        tmem_wait_ld(d[1]);
        const uint32_t stat = sbase + kSmStat + (n & 1) * kStatBytes + kTile * 4 + wg * 256;
        const uint64_t neg2 = f2_pack(neg_delta, neg_delta);
        const uint32_t tDs = kDq ? tT1 : tT2;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            uint64_t la = neg2, lb = neg2;
            if (!kDq) lds_f2x2(stat + (c * 32 + e * 2) * 4, la, lb);
            w[e] = pack_pair(f2_mul(pr[c * 16 + e], f2_add(f2_pack(u2f(d[c][2 * e]), u2f(d[c][2 * e + 1])), la)));
            w[e + 1] = pack_pair(
                f2_mul(pr[c * 16 + e + 1], f2_add(f2_pack(u2f(d[c][2 * e + 2]), u2f(d[c][2 * e + 3])), lb)));
          }
          tmem_st16(tDs + c * 16, w);
        }
      }
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      named_bar_arrive(kBarDs, kSoftmaxThreads + 32);
      ++n;
    }
  } else if (warp < kProducerWarp) {
    regs_decrease<kBwdRegsEpi>();
    // ------------------------------------------------------------ epilogue
    const int row = threadIdx.x & 127;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const int rows = kDq ? p.seq_q : p.seq_kv;
    bool ok = true;
    uint32_t done = 0;  // items with tiles so far
    Items<kDq> it(p);
    while (it.next()) {
      const int r = it.tile * kTile + row;
      const bool write = r < rows;
      const long long at = (static_cast<long long>(it.head) * rows + r) * kHeadDim;
      // dK/dV: dV (accumulator 2, complete first), then dK; dQ: accumulator 1 only.
#pragma unroll 1
      for (int a = kDq ? 1 : 2; a >= 1; --a) {
        __nv_bfloat16* const dst = static_cast<__nv_bfloat16*>(a == 1 ? p.g1 : p.g2) + at;
        const float f = a == 1 ? p.scale : 1.f;
        const uint32_t acc = tmem + lane_off + (a == 1 ? kColAcc1 : kColAcc2);
        if (it.n > 0 && ok) {
          ok = __all_sync(0xffffffffu, wait_phase(bar(a == 1 ? B_ACC1 : B_ACC2), done & 1, watch));
          tc_fence_after();
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32];
          if (it.n > 0 && ok) {
            tmem_ld32(acc + c * 32, o);
            tmem_wait_ld(o);
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0u;
          }
          if (c == 3 && it.n > 0) {
            // Read out: the next item may overwrite it.
            tc_fence_before();
            __syncwarp();
            if (ok)
              named_bar_arrive(a == 1 ? kBarAcc1 : kBarAcc2, 128 + 32);
            else
              named_bar_sync(a == 1 ? kBarAcc1 : kBarAcc2, 128 + 32);
          }
          if (write && ok) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              uint32_t w[8];
#pragma unroll
              for (int e = 0; e < 8; ++e)
                w[e] = pack_bf16x2(u2f(o[16 * q + 2 * e]) * f, u2f(o[16 * q + 2 * e + 1]) * f);
              st_global_v8(dst + c * 32 + q * 16, w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]);
            }
          }
        }
      }
      if (it.n > 0) ++done;
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
      // Waits until a buffer's last user is done and its previous copy has landed (the
      // latter is implied unless the CTA aborted): at most one copy per buffer in flight.
      auto reuse = [&](int empty, int full, uint32_t parity) {
        return wait_phase(bar(empty), parity, watch) && wait_phase(bar(full), parity, watch) && !*abort_flag;
      };
      int n = 0, items = 0, n2 = 0, nx2 = 0, nst = 0, skipped = -1;
      Tiles<kDq> it(p);
      while (it.next()) {
        const int s1 = n % kY1, s2 = n % kY2;
        if (n >= kY1 && !reuse(B_Y1_EMPTY + s1, B_Y1_FULL + s1, (n / kY1 - 1) & 1)) break;
        if (*abort_flag) break;
        if (n == p.test_skip_load) skipped = n;  // test hook: this copy never arrives
        if (n != skipped) load(kSmY1 + s1 * kTileBytes, &tm_y1, B_Y1_FULL + s1, it.t * kTile, it.y_head, pol_y);
        ++n;
        if (it.first) {
          if (items > 0 && !reuse(B_X1_EMPTY, B_X1_FULL, (items - 1) & 1)) break;
          load(kSmX1, &tm_x1, B_X1_FULL, it.items.tile * kTile, it.items.head, pol_x);
          ++items;
        }
        if (n2 >= kY2 && !reuse(B_Y2_EMPTY + s2, B_Y2_FULL + s2, (n2 / kY2 - 1) & 1)) break;
        load(kSmY2 + s2 * kTileBytes, &tm_y2, B_Y2_FULL + s2, it.t * kTile, it.y_head, pol_y);
        ++n2;
        if (it.first) {
          if (nx2 > 0 && !reuse(B_X2_EMPTY, B_X2_FULL, (nx2 - 1) & 1)) break;
          load(kSmX2, &tm_x2, B_X2_FULL, it.items.tile * kTile, it.items.head, pol_x);
          ++nx2;
        }
        if (!kDq) {
          // The slot's last readers published dS of tile nst - 2 before that tile's dK MMAs,
          // whose completion empties its Y1 slot.
          const int u = nst - 2;
          if (u >= 0 && !(wait_phase(bar(B_Y1_EMPTY + u % kY1), (u / kY1) & 1, watch) &&
                          wait_phase(bar(B_STAT + (u & 1)), (u >> 1) & 1, watch) && !*abort_flag))
            break;
          const float* src = p.stats + (static_cast<long long>(it.y_head) * p.nq + it.t) * (2 * kTile);
          mbar_arrive_expect_tx(bar(B_STAT + (nst & 1)), kStatBytes);
          bulk_load(sbase + kSmStat + (nst & 1) * kStatBytes, src, kStatBytes, bar(B_STAT + (nst & 1)));
          ++nst;
        }
      }
      if (*abort_flag) {
        // Copies already issued still land in shared memory: wait for them.
        for (int u = max(0, n - kY1); u < n; ++u)
          if (u != skipped) drain_phase(bar(B_Y1_FULL + u % kY1), (u / kY1) & 1, watch);
        for (int u = max(0, n2 - kY2); u < n2; ++u) drain_phase(bar(B_Y2_FULL + u % kY2), (u / kY2) & 1, watch);
        for (int u = max(0, nst - 2); u < nst; ++u) drain_phase(bar(B_STAT + (u & 1)), (u >> 1) & 1, watch);
        if (items > 0) drain_phase(bar(B_X1_FULL), (items - 1) & 1, watch);
        if (nx2 > 0) drain_phase(bar(B_X2_FULL), (nx2 - 1) & 1, watch);
      }
    }
    __syncwarp();
  } else if (warp == kIssuerWarp) {
    regs_decrease<kBwdRegsOther>();
    // ------------------------------------------------------------ MMA issuer
    const bool leader = lane == 0;
    const uint32_t tT1 = tmem + kColT1, tT2 = tmem + kColT2, tA1 = tmem + kColAcc1, tA2 = tmem + kColAcc2;
    const uint32_t x1 = smem_desc_lo(sbase + kSmX1, 16), x2 = smem_desc_lo(sbase + kSmX2, 16);
    // Streamed tiles as the N x K operand of T1 and T2, and as the K x N operand of the
    // accumulating MMAs.
    const uint32_t y1 = smem_desc_lo(sbase + kSmY1, 16), y1t = smem_desc_lo(sbase + kSmY1, kHalfBytes);
    const uint32_t y2 = smem_desc_lo(sbase + kSmY2, 16), y2t = smem_desc_lo(sbase + kSmY2, kHalfBytes);
    constexpr uint32_t kSlot = kTileBytes >> 4;
    auto sync_on = [&](uint32_t id, uint32_t threads) {
      __syncwarp();
      named_bar_sync(id, threads);
      tc_fence_after();
    };
    Tiles<kDq> it(p);
    uint32_t items = 0;
    if constexpr (!kDq) {
      bool have = it.next();
      int s1 = 0, s2 = 0;  // slots of the current tile
      if (have) {
        sync_on(kBarLoaded, 64);
        if (leader) {
          issue_xy(tT1, x1, y1);
          mma_commit(bar(B_T1_FULL));
          if (it.last) mma_commit(bar(B_X1_EMPTY));
        }
        sync_on(kBarLoaded, 64);
        if (leader) {
          issue_xy(tT2, x2, y2);
          mma_commit(bar(B_T2_FULL));
          if (it.last) mma_commit(bar(B_X2_EMPTY));
        }
      }
      while (have) {
        const bool first = it.first, last = it.last;
        const bool more = it.next();
        const bool next_last = more && it.last;
        const int n1 = s1 == kY1 - 1 ? 0 : s1 + 1, n2 = s2 ^ 1;
        if (first && items > 0) sync_on(kBarAcc2, 128 + 32);
        sync_on(kBarP, kSoftmaxThreads + 32);
        if (leader) {
          issue_acc(tA2, tT1, y2t + s2 * kSlot, first ? 0u : 1u);
          mma_commit(bar(B_Y2_EMPTY + s2));
          if (last) mma_commit(bar(B_ACC2));
        }
        if (more) {
          sync_on(kBarLoaded, 64);
          if (leader) {
            issue_xy(tT1, x1, y1 + n1 * kSlot);
            mma_commit(bar(B_T1_FULL));
            if (next_last) mma_commit(bar(B_X1_EMPTY));
          }
        }
        if (first && items > 0) sync_on(kBarAcc1, 128 + 32);
        sync_on(kBarDs, kSoftmaxThreads + 32);
        if (leader) {
          issue_acc(tA1, tT2, y1t + s1 * kSlot, first ? 0u : 1u);
          mma_commit(bar(B_Y1_EMPTY + s1));
          if (last) mma_commit(bar(B_ACC1));
        }
        if (more) {
          sync_on(kBarLoaded, 64);
          if (leader) {
            issue_xy(tT2, x2, y2 + n2 * kSlot);
            mma_commit(bar(B_T2_FULL));
            if (next_last) mma_commit(bar(B_X2_EMPTY));
          }
        }
        if (first) ++items;
        s1 = n1;
        s2 = n2;
        have = more;
      }
      if (items > 0) {
        sync_on(kBarAcc2, 128 + 32);
        sync_on(kBarAcc1, 128 + 32);
      }
    } else {
      // S runs two tiles ahead (T1 | acc2 columns are its two buffers), dP one.
      bool f0 = false, l0 = false, f1 = false, l1 = false;
      bool have = it.next(), have1 = false;
      if (have) {
        f0 = it.first;
        l0 = it.last;
        sync_on(kBarLoaded, 64);
        if (leader) {
          issue_xy(tT1, x1, y1);
          mma_commit(bar(B_T1_FULL));
          if (l0) mma_commit(bar(B_X1_EMPTY));
        }
        sync_on(kBarLoaded, 64);
        if (leader) {
          issue_xy(tT2, x2, y2);
          mma_commit(bar(B_T2_FULL));
          mma_commit(bar(B_Y2_EMPTY));
          if (l0) mma_commit(bar(B_X2_EMPTY));
        }
        have1 = it.next();
        f1 = it.first;
        l1 = it.last;
        if (have1) {
          sync_on(kBarLoaded, 64);
          if (leader) {
            issue_xy(tA2, x1, y1 + kSlot);
            mma_commit(bar(B_T1_FULL + 1));
            if (l1) mma_commit(bar(B_X1_EMPTY));
          }
        }
      }
      int s1 = 0, par = 0;
      while (have) {
        const bool have2 = have1 && it.next();
        const bool f2 = it.first, l2 = it.last;
        const int s1_2 = s1 == 0 ? 2 : s1 - 1;  // slot of tile n + 2
        const uint32_t tS = par ? tA2 : tT1;
        sync_on(kBarDs, kSoftmaxThreads + 32);
        if (have1) {
          sync_on(kBarLoaded, 64);
          if (leader) {
            issue_xy(tT2, x2, y2 + (par ^ 1) * kSlot);
            mma_commit(bar(B_T2_FULL));
            mma_commit(bar(B_Y2_EMPTY + (par ^ 1)));
            if (l1) mma_commit(bar(B_X2_EMPTY));
          }
        }
        if (f0 && items > 0) sync_on(kBarAcc1, 128 + 32);
        if (leader) {
          issue_acc(tA1, tS, y1t + s1 * kSlot, f0 ? 0u : 1u);
          mma_commit(bar(B_Y1_EMPTY + s1));
          if (l0) mma_commit(bar(B_ACC1));
        }
        if (have2) {
          sync_on(kBarLoaded, 64);
          if (leader) {
            issue_xy(tS, x1, y1 + s1_2 * kSlot);
            mma_commit(bar(B_T1_FULL + par));
            if (l2) mma_commit(bar(B_X1_EMPTY));
          }
        }
        if (f0) ++items;
        f0 = f1;
        l0 = l1;
        f1 = f2;
        l1 = l2;
        have = have1;
        have1 = have2;
        s1 = s1 == kY1 - 1 ? 0 : s1 + 1;
        par ^= 1;
      }
      if (items > 0) sync_on(kBarAcc1, 128 + 32);
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
    // The loads' mbarrier waits in the issuer's order: X1 and Y1 of a tile for T1, X2 and Y2
    // for T2.  After an abort the waits return at once and only the rounds are kept.
    int n = 0, items = 0;
    Tiles<kDq> it(p);
    while (it.next()) {
      if (lane == 0) {
        if (it.first) wait_phase(bar(B_X1_FULL), items & 1, watch);
        wait_phase(bar(B_Y1_FULL + n % kY1), (n / kY1) & 1, watch);
      }
      __syncwarp();
      named_bar_sync(kBarLoaded, 64);
      if (lane == 0) {
        if (it.first) wait_phase(bar(B_X2_FULL), items & 1, watch);
        wait_phase(bar(B_Y2_FULL + n % kY2), (n / kY2) & 1, watch);
      }
      __syncwarp();
      named_bar_sync(kBarLoaded, 64);
      if (it.first) ++items;
      ++n;
    }
  } else {
    regs_decrease<kBwdRegsOther>();  // warp 15 completes the warpgroup
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kIssuerWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
  // The dQ launch is complete only when the dK/dV launch is (see above).
  if (kDq) grid_dependency_wait();
}

// -LSE*log2(e) and -delta of every query row, padded to whole tiles: [heads][nq][2][128].
// 16 lanes per row, 16 bytes of O and dO each.  Rows past seq_q and rows that saw no key
// (LSE = -inf) get -inf, so their probabilities are exactly 0.
__global__ void __launch_bounds__(256)
    stats_kernel(const uint4* __restrict__ dout, const uint4* __restrict__ out, const float* __restrict__ lse,
                 float* __restrict__ stats, long long rows_padded, int seq_q, int nq) {
  grid_dependency_wait();
  grid_launch_dependents();
  const long long g = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 4;
  const int l = threadIdx.x & 15;
  if (g >= rows_padded) return;  // whole warps: rows_padded is a multiple of 128
  const long long tile = g >> 7;
  const int r = static_cast<int>(g & 127);
  const long long head = tile / nq;
  const int row = static_cast<int>(tile % nq) * kTile + r;
  float acc = 0.f;
  if (row < seq_q) {
    const long long at = (head * seq_q + row) * 16 + l;
    const uint4 a = dout[at], b = out[at];
    const uint32_t wa[4] = {a.x, a.y, a.z, a.w}, wb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      acc = fmaf(u2f(wa[i] << 16), u2f(wb[i] << 16), acc);
      acc = fmaf(u2f(wa[i] & 0xffff0000u), u2f(wb[i] & 0xffff0000u), acc);
    }
  }
#pragma unroll
  for (int m = 8; m > 0; m >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, m);
  if (l == 0) {
    float neg = -CUDART_INF_F;
    if (row < seq_q) {
      const float v = lse[head * seq_q + row];
      neg = v == -CUDART_INF_F ? v : -v * 1.4426950408889634f;
    }
    float* dst = stats + tile * (2 * kTile) + r;
    dst[0] = neg;
    dst[kTile] = -acc;
  }
}

}  // namespace bwd
}  // namespace avo_b200
