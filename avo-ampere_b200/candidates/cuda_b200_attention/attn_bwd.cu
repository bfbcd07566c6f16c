// C-ABI entry points of the attention gradient (declared in include/avo_b200_attn.h): argument checks, tensor maps
// and the launches of attn_bwd.cuh.
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>

#include "attn_bwd.cuh"
#include "avo_b200_attn.h"
#include "host_common.h"

namespace avo_b200 {
namespace {

using bwd::kTile;

int tiles_of(int rows) { return rows / kTile + (rows % kTile != 0); }

template <bool kDq>
auto kernel_of(bwd::Order order) {
  return order == bwd::kPairs     ? bwd::attn_bwd_kernel<kDq, bwd::kPairs>
         : order == bwd::kLongest ? bwd::attn_bwd_kernel<kDq, bwd::kLongest>
         : order == bwd::kEqual   ? bwd::attn_bwd_kernel<kDq, bwd::kEqual>
                                  : bwd::attn_bwd_kernel<kDq, bwd::kAny>;
}

// The kernels' shared-memory limit and register allocation, once per device.
int prepare_bwd(int* sm_count) {
  const int rc = host::device(sm_count);
  if (rc != AVO_B200_OK) return rc;
  static std::atomic<int> ready[64];
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0) {
    (void)cudaGetLastError();
    return AVO_B200_ENODEV;
  }
  if (dev < 64 && ready[dev].load(std::memory_order_acquire) == 1) return AVO_B200_OK;
  const void* kernels[] = {reinterpret_cast<const void*>(kernel_of<false>(bwd::kAny)),
                           reinterpret_cast<const void*>(kernel_of<true>(bwd::kAny)),
                           reinterpret_cast<const void*>(kernel_of<false>(bwd::kEqual)),
                           reinterpret_cast<const void*>(kernel_of<true>(bwd::kEqual)),
                           reinterpret_cast<const void*>(kernel_of<false>(bwd::kLongest)),
                           reinterpret_cast<const void*>(kernel_of<true>(bwd::kLongest)),
                           reinterpret_cast<const void*>(kernel_of<false>(bwd::kPairs)),
                           reinterpret_cast<const void*>(kernel_of<true>(bwd::kPairs))};
  for (const void* k : kernels) {
    cudaFuncAttributes attr{};
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, bwd::kBwdSmemBytes) != cudaSuccess ||
        cudaFuncGetAttributes(&attr, k) != cudaSuccess) {
      (void)cudaGetLastError();
      return AVO_B200_ELAUNCH;
    }
    // The setmaxnreg split only works out with the allocation it was computed for.
    if (attr.numRegs != static_cast<int>(bwd::kBwdRegsLaunch)) return AVO_B200_EREGS;
  }
  if (dev < 64) ready[dev].store(1, std::memory_order_release);
  return AVO_B200_OK;
}

bool sizes_ok(int batch, int heads, int kv_heads, int seq_q, int seq_kv) {
  if (batch < 0 || heads < 0 || kv_heads <= 0 || seq_q < 0 || seq_kv < 0 || heads % kv_heads != 0) return false;
  if (seq_q > INT_MAX - 2 * kTile || seq_kv > INT_MAX - 2 * kTile) return false;
  const long long qh = static_cast<long long>(batch) * heads;
  if (qh > INT_MAX) return false;
  // Work items, and the tiles of one item over its group of heads, are counted in ints.
  const long long nq = tiles_of(seq_q), nkv = tiles_of(seq_kv);
  return qh * nq <= INT_MAX && qh * nkv <= INT_MAX && (heads / kv_heads) * nq <= INT_MAX;
}

// Without a mask, and for a single query, the rows of the query heads that share a key/value
// head attend alike, and they are adjacent in memory: one head of group * seq_q rows.  Fewer
// partly filled tiles (and none of the group's heads reads the keys again).
void fold_group(int& heads, int kv_heads, int& seq_q, int seq_kv, int& causal) {
  if (seq_q == 1 && seq_kv > 0) causal = 0;  // the last query sees every key
  const long long rows = static_cast<long long>(heads / kv_heads) * seq_q;
  if (causal || rows > INT_MAX - 2 * kTile) return;
  seq_q = static_cast<int>(rows);
  heads = kv_heads;
}

// What a call runs, from its sizes alone (of a B200's 148 multiprocessors, so that neither the
// scratch nor the results depend on the device that happens to be current).
struct Sizes {
  int q_heads, kv_heads, group;  // batch * heads
  int seq_q, seq_kv, nq, nkv;
  int causal, offset;
  int split_kv, split_q;         // pieces per item of the dK/dV and of the dQ pass
  size_t part_kv, part_q;        // bytes of one gradient's partial sums (dK or dV; dQ)
};
constexpr int kPlanSms = 148;

// Pieces per item of both passes.  In microseconds: a tile takes about 1.4 (dK/dV) or 1.2 (dQ),
// a unit's start and end five tiles more; a join about 4 and its bytes at 3 TB/s.  Units of both
// passes that fit the chip all at once take as long as the longest.  Otherwise a dK/dV that
// fills the chip comes first; one that does not leaves gaps, where units of dQ start early, but
// CTAs with several of them have as many wherever they start.  One piece unless more win a
// twentieth.  Measured on B200, one piece against the pieces chosen here (dK/dV, dQ): B1 H8
// Hkv2 S2048 causal 92 / 42 us (4, 1), B1 H16 Hkv2 Q300 KV2048 causal 50 / 36 (2, 1), B1 H1
// S4096 52 / 39 (2, 2), B1 H32 Hkv4 S2048 causal 217 / 117 (4, 1); but B1 H12 S1000 34 us,
// with (2, 1) 38.
void choose_split(Sizes& z, double kv_items, double kv_longest, double q_items, double q_longest, double total) {
  static constexpr int kPieces[] = {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 16, 20, 24, 28, 32};
  z.split_kv = z.split_q = 1;
  // (32 pieces keep every product of a tile count and a piece within 32 bits.)
  if (std::max(kv_longest, q_longest) * 32 > INT_MAX || std::max(kv_items, q_items) * 32 > INT_MAX) return;
  double best = 0.0;
  for (const int kv : kPieces) {
    const double kv_units = kv_items * kv;
    if (kv > 1 && (kv > kv_longest || kv_units > 3 * kPlanSms)) break;
    const double kv_us = 1.4 * (std::ceil(kv_longest / kv) + 5.0), kv_all = 1.4 * (total + 5.0 * kv_units);
    for (const int q : kPieces) {
      const double q_units = q_items * q;
      if (q > 1 && (q > q_longest || q_units > 3 * kPlanSms)) break;
      const double q_us = 1.2 * (std::ceil(q_longest / q) + 5.0), q_all = 1.2 * (total + 5.0 * q_units);
      double us = std::max(kv_us, q_us);
      if (kv_units + q_units > kPlanSms) {
        if (kv_units >= kPlanSms) {
          // (Units of different lengths make up for one another, equal ones do not.)
          const bool equal = q_items * q_longest <= 1.1 * total;
          const double q_turns = equal ? std::ceil(q_units / kPlanSms) * q_us : q_all / kPlanSms;
          us = std::max(kv_us, kv_all / kPlanSms) + std::max(q_us, q_turns);
        } else {
          // (No more units of dQ then: beside dK/dV they would take up to twice as long.)
          if (q > 1) break;
          us = std::max({us, (kv_all + q_all) / kPlanSms, std::min(kv_all / kv_units, q_all / q_units) + q_all / q_units});
          if (q_units > kPlanSms) us = std::max(us, kv_us + q_all / kPlanSms);
        }
      }
      if (kv > 1 || q > 1) us += 4.0;
      if (kv > 1) us += kv * 2.0 * z.part_kv / 3e6;
      if (q > 1) us += q * 1.0 * z.part_q / 3e6;
      if (kv == 1 && q == 1) {
        best = 0.95 * us;
      } else if (us < best) {
        best = us;
        z.split_kv = kv;
        z.split_q = q;
      }
    }
  }
}

Sizes sizes_of(int batch, int heads, int kv_heads, int seq_q, int seq_kv, int causal) {
  Sizes z{};
  fold_group(heads, kv_heads, seq_q, seq_kv, causal);
  z.q_heads = batch * heads;
  z.kv_heads = batch * kv_heads;
  z.group = heads / kv_heads;
  z.seq_q = seq_q;
  z.seq_kv = seq_kv;
  z.nq = tiles_of(seq_q);
  z.nkv = tiles_of(seq_kv);
  z.causal = causal ? 1 : 0;
  z.offset = causal ? seq_kv - seq_q : 0;
  z.part_kv = static_cast<size_t>(z.kv_heads) * seq_kv * kHeadDim * sizeof(float);
  z.part_q = static_cast<size_t>(z.q_heads) * seq_q * kHeadDim * sizeof(float);
  if (z.part_kv == 0 || z.part_q == 0) {
    z.split_kv = z.split_q = 1;
    return z;
  }
  // Tiles that some row needs, of nq * nkv per query head: with a mask, about the visible pairs
  // and half of the diagonal's tiles.
  double pairs = static_cast<double>(z.nq) * z.nkv;
  if (z.causal) {
    const double rows = std::min(seq_q, seq_kv);  // rows that see a key
    const double seen = rows * std::max(0, seq_kv - seq_q) + rows * (rows + 1.0) / 2.0;
    pairs = std::min(pairs, seen / (kTile * kTile) + 0.5 * tiles_of(std::min(seq_q, seq_kv)));
  }
  const double kv_items = static_cast<double>(z.kv_heads) * z.nkv, q_items = static_cast<double>(z.q_heads) * z.nq;
  choose_split(z, kv_items, static_cast<double>(z.group) * z.nq, q_items, z.nkv, pairs * z.q_heads);
  return z;
}

size_t round256(size_t x) { return (x + 255) / 256 * 256; }

// Causal items are taken in pairs where whole pairs leave less than a twentieth of the
// multiprocessors' time idle.  Longest first balances any number of items, but has all heads in
// flight at once: where they do not fit L2 they are read from memory again and again, and that
// takes power from the multiprocessors' clock (measured on B200, longest first against pairs,
// back to back at the power limit: B8 H16 S2048 590 us at 1.17 GHz / 525 at 1.45, B2 H16 S8192
// 1690 / 1590, B16 H16 S1024 383 / 350; but B1 H16 S4096, 1.7 pairs to a multiprocessor,
// 220 / 240).
bwd::Order order_of(const Sizes& z, int sms) {
  if (z.split_kv > 1 || z.split_q > 1) return bwd::kAny;
  if (!z.causal) return bwd::kEqual;
  if (z.offset != 0) return bwd::kAny;
  const long long kv = z.kv_heads * ((z.nkv + 1LL) / 2), q = z.q_heads * ((z.nq + 1LL) / 2);
  const double kv_us = 1.4 * (z.group * (z.nq + 1.0) + 10.0), q_us = 1.2 * (z.nkv + 1.0 + 10.0);
  // Multiprocessors with one pair more of dK/dV are the last to have one more of dQ.
  const long long kv_more = kv % sms, q_more = q % sms;
  double most = kv_more + q_more > sms ? kv_us + q_us : std::max(kv_more > 0 ? kv_us : 0.0, q_more > 0 ? q_us : 0.0);
  most += kv / sms * kv_us + q / sms * q_us;
  return most * 0.95 * sms < kv * kv_us + q * q_us ? bwd::kPairs : bwd::kLongest;
}

void set_items(bwd::BwdParams& p, int heads, int tiles, int split, bwd::Order order) {
  p.split = static_cast<uint32_t>(split);
  p.split_magic = ~0ull / p.split + 1;  // unused for 1
  const int rows = order == bwd::kPairs ? (tiles + 1) / 2 : tiles;
  p.item_count = static_cast<uint32_t>(heads) * static_cast<uint32_t>(rows) * p.split;
  p.item_div = static_cast<uint32_t>(p.causal && order != bwd::kPairs ? heads : rows);
  p.item_magic = ~0ull / p.item_div + 1;
}

constexpr size_t kClaimBytes = 2 * bwd::kMaxClaims * sizeof(uint32_t);

// Claims and row statistics.
size_t stats_bytes(const Sizes& z) {
  return round256(static_cast<size_t>(z.q_heads) * z.nq * bwd::kStatBytes + kClaimBytes);
}

size_t scratch_bytes(const Sizes& z) {
  return stats_bytes(z) + (z.split_kv > 1 ? 2 * z.split_kv * z.part_kv : 0) + (z.split_q > 1 ? z.split_q * z.part_q : 0);
}

int zero(void* p, size_t bytes, cudaStream_t st) {
  if (bytes == 0) return AVO_B200_OK;
  if (p == nullptr) return AVO_B200_EINVAL;
  if (cudaMemsetAsync(p, 0, bytes, st) == cudaSuccess) return AVO_B200_OK;
  (void)cudaGetLastError();
  return AVO_B200_ELAUNCH;
}

}  // namespace
}  // namespace avo_b200

using namespace avo_b200;

extern "C" int avo_b200_attn_bwd_workspace_size(int batch, int heads, int kv_heads, int seq_q, int seq_kv,
                                                int causal, size_t* bytes) {
  if (bytes == nullptr || !sizes_ok(batch, heads, kv_heads, seq_q, seq_kv)) return AVO_B200_EINVAL;
  *bytes = scratch_bytes(sizes_of(batch, heads, kv_heads, seq_q, seq_kv, causal));
  return AVO_B200_OK;
}

extern "C" int avo_b200_attn_bwd(const void* dout, const void* q, const void* k, const void* v, const void* out,
                                 const float* lse, void* dq, void* dk, void* dv, int batch, int heads, int kv_heads,
                                 int seq_q, int seq_kv, int head_dim, int causal, float softmax_scale,
                                 void* workspace, size_t workspace_bytes, int* status_dev, void* stream) {
  if (head_dim != kHeadDim || !sizes_ok(batch, heads, kv_heads, seq_q, seq_kv)) return AVO_B200_EINVAL;
  if (!(softmax_scale > 0.f) || !std::isfinite(softmax_scale)) return AVO_B200_EINVAL;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Sizes z = sizes_of(batch, heads, kv_heads, seq_q, seq_kv, causal);
  const size_t q_bytes = z.part_q / 2, kv_bytes = z.part_kv / 2;
  if (q_bytes == 0 || kv_bytes == 0) {
    // Nothing attends to anything: whichever gradients exist are zero.
    int rc = zero(dq, q_bytes, st);
    if (rc == AVO_B200_OK) rc = zero(dk, kv_bytes, st);
    if (rc == AVO_B200_OK) rc = zero(dv, kv_bytes, st);
    return rc;
  }
  const void* inputs[] = {dout, q, k, v, out};
  for (const void* p : inputs)
    if (p == nullptr || !host::aligned(p, 16)) return AVO_B200_EINVAL;
  void* const grads[] = {dq, dk, dv};
  for (void* p : grads)
    if (p == nullptr || !host::aligned(p, 32)) return AVO_B200_EINVAL;
  if (lse == nullptr || !host::aligned(lse, 4)) return AVO_B200_EINVAL;
  if (workspace == nullptr || !host::aligned(workspace, 256) || workspace_bytes < scratch_bytes(z))
    return AVO_B200_EINVAL;

  int sms = 0;
  int rc = prepare_bwd(&sms);
  if (rc != AVO_B200_OK) return rc;
  alignas(64) CUtensorMap tq, tk, tv, tdo;
  if ((rc = host::encode(&tq, q, z.seq_q, z.q_heads)) != AVO_B200_OK) return rc;
  if ((rc = host::encode(&tdo, dout, z.seq_q, z.q_heads)) != AVO_B200_OK) return rc;
  if ((rc = host::encode(&tk, k, z.seq_kv, z.kv_heads)) != AVO_B200_OK) return rc;
  if ((rc = host::encode(&tv, v, z.seq_kv, z.kv_heads)) != AVO_B200_OK) return rc;

  bwd::BwdParams p{};
  uint32_t* const claims = static_cast<uint32_t*>(workspace);
  float* const stats = reinterpret_cast<float*>(static_cast<char*>(workspace) + kClaimBytes);
  p.stats = stats;
  p.status = status_dev;
  p.watchdog_ns = host::watchdog_limit();
  p.seq_q = z.seq_q;
  p.seq_kv = z.seq_kv;
  p.nq = z.nq;
  p.nkv = z.nkv;
  p.q_heads = z.q_heads;
  p.kv_heads = z.kv_heads;
  p.group = z.group;
  p.causal = z.causal;
  p.offset = z.offset;
  p.scale = softmax_scale;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.test_skip_load = host::skip_load();
  float* const part_dk = reinterpret_cast<float*>(static_cast<char*>(workspace) + stats_bytes(z));
  float* const part_dv = part_dk + (z.split_kv > 1 ? z.split_kv * z.part_kv / sizeof(float) : 0);
  float* const part_dq = part_dv + (z.split_kv > 1 ? z.split_kv * z.part_kv / sizeof(float) : 0);

  const bwd::Order order = order_of(z, sms);
  const long long kv_units = static_cast<long long>(z.kv_heads) * z.nkv * z.split_kv;
  const long long q_units = static_cast<long long>(z.q_heads) * z.nq * z.split_q;
  // With a unit for every multiprocessor, CTAs take them by place (see the kernel).  Not with
  // fewer: the two passes then share the chip from the start, and CTAs without a unit would
  // leave their places to later ones on the same multiprocessor (measured on B200, B1 H8 S2048,
  // 128 units a pass: 54 us, with places and idle CTAs 110).
  const bool by_place = kv_units >= sms && sms <= bwd::kMaxClaims;
  const unsigned kv_grid = static_cast<unsigned>(kv_units > sms ? sms : kv_units);
  const unsigned q_grid = static_cast<unsigned>(q_units > sms ? sms : q_units);

  const long long blocks = static_cast<long long>(z.q_heads) * p.nq * (kTile / bwd::kStatBlockRows);
  if (blocks > INT_MAX) return AVO_B200_EINVAL;
  if (!host::launch_early(bwd::stats_kernel, static_cast<unsigned>(blocks), 256u, 0, st,
                          static_cast<const uint4*>(dout), static_cast<const uint4*>(out), lse, stats, z.seq_q, p.nq,
                          claims))
    return AVO_B200_ELAUNCH;
  set_items(p, z.kv_heads, z.nkv, z.split_kv, order);
  p.claims = by_place ? claims : nullptr;
  p.g1 = dk;
  p.g2 = dv;
  p.part1 = part_dk;
  p.part2 = part_dv;
  if (!host::launch_early(kernel_of<false>(order), kv_grid, bwd::kBwdThreads, bwd::kBwdSmemBytes, st, tk, tv, tq, tdo, p))
    return AVO_B200_ELAUNCH;
  set_items(p, z.q_heads, z.nq, z.split_q, order);
  p.claims = by_place && q_units >= sms ? claims + bwd::kMaxClaims : nullptr;
  p.g1 = dq;
  p.g2 = nullptr;
  p.part1 = part_dq;
  p.x1 = q;
  if (!host::launch_early(kernel_of<true>(order), q_grid, bwd::kBwdThreads, bwd::kBwdSmemBytes, st, tq, tdo, tk, tv, p))
    return AVO_B200_ELAUNCH;
  if (z.split_kv > 1 || z.split_q > 1) {
    bwd::JoinParams j{};
    void* const out[3] = {dk, dv, dq};
    const float* const part[3] = {part_dk, part_dv, part_dq};
    long long groups = 0;
    for (int g = 0; g < 3; ++g) {
      const int split = g < 2 ? z.split_kv : z.split_q;
      j.part[g] = part[g];
      j.out[g] = static_cast<__nv_bfloat16*>(out[g]);
      j.factor[g] = g == 1 ? 1.f : softmax_scale;
      j.pieces[g] = static_cast<uint32_t>(split);
      j.count[g] = split > 1 ? static_cast<long long>((g < 2 ? z.part_kv : z.part_q) / (8 * sizeof(float))) : 0;
      groups += j.count[g];
    }
    if (!host::launch_early(bwd::join_kernel, static_cast<unsigned>((groups + 255) / 256), 256u, 0, st, j))
      return AVO_B200_ELAUNCH;
  }
  return cudaGetLastError() == cudaSuccess ? AVO_B200_OK : AVO_B200_ELAUNCH;
}
