// C-ABI entry points of the attention gradient (declared in include/avo_b200_attn.h): argument checks, tensor maps
// and the three launches of attn_bwd.cuh.
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
  const void* kernels[] = {reinterpret_cast<const void*>(bwd::attn_bwd_kernel<false>),
                           reinterpret_cast<const void*>(bwd::attn_bwd_kernel<true>)};
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

size_t stats_bytes(int batch, int heads, int seq_q) {
  return static_cast<size_t>(batch) * heads * tiles_of(seq_q) * bwd::kStatBytes;
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
                                                size_t* bytes) {
  if (bytes == nullptr || !sizes_ok(batch, heads, kv_heads, seq_q, seq_kv)) return AVO_B200_EINVAL;
  *bytes = stats_bytes(batch, heads, seq_q);  // not less than with the group folded
  return AVO_B200_OK;
}

extern "C" int avo_b200_attn_bwd(const void* dout, const void* q, const void* k, const void* v, const void* out,
                                 const float* lse, void* dq, void* dk, void* dv, int batch, int heads, int kv_heads,
                                 int seq_q, int seq_kv, int head_dim, int causal, float softmax_scale,
                                 void* workspace, size_t workspace_bytes, int* status_dev, void* stream) {
  if (head_dim != kHeadDim || !sizes_ok(batch, heads, kv_heads, seq_q, seq_kv)) return AVO_B200_EINVAL;
  if (!(softmax_scale > 0.f) || !std::isfinite(softmax_scale)) return AVO_B200_EINVAL;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t wanted = stats_bytes(batch, heads, seq_q);
  fold_group(heads, kv_heads, seq_q, seq_kv, causal);
  const int q_heads = batch * heads, kv_all = batch * kv_heads;
  const size_t q_bytes = static_cast<size_t>(q_heads) * seq_q * kHeadDim * 2;
  const size_t kv_bytes = static_cast<size_t>(kv_all) * seq_kv * kHeadDim * 2;
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
  if (workspace == nullptr || !host::aligned(workspace, 256) || workspace_bytes < wanted)
    return AVO_B200_EINVAL;

  int sms = 0;
  int rc = prepare_bwd(&sms);
  if (rc != AVO_B200_OK) return rc;
  alignas(64) CUtensorMap tq, tk, tv, tdo;
  if ((rc = host::encode(&tq, q, seq_q, q_heads)) != AVO_B200_OK) return rc;
  if ((rc = host::encode(&tdo, dout, seq_q, q_heads)) != AVO_B200_OK) return rc;
  if ((rc = host::encode(&tk, k, seq_kv, kv_all)) != AVO_B200_OK) return rc;
  if ((rc = host::encode(&tv, v, seq_kv, kv_all)) != AVO_B200_OK) return rc;

  bwd::BwdParams p{};
  p.stats = static_cast<const float*>(workspace);
  p.status = status_dev;
  p.watchdog_ns = host::watchdog_limit();
  p.seq_q = seq_q;
  p.seq_kv = seq_kv;
  p.nq = tiles_of(seq_q);
  p.nkv = tiles_of(seq_kv);
  p.q_heads = q_heads;
  p.kv_heads = kv_all;
  p.group = heads / kv_heads;
  p.causal = causal ? 1 : 0;
  p.offset = causal ? seq_kv - seq_q : 0;
  p.scale = softmax_scale;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.test_skip_load = host::skip_load();

  const long long kv_items = static_cast<long long>(kv_all) * p.nkv, q_items = static_cast<long long>(q_heads) * p.nq;
  // Both passes at once where the dK/dV grid leaves multiprocessors idle from the start.
  // Measured on B200, at once against one after the other: B1 H4 S512 14.1 / 22.9 us, B1 H16
  // Hkv2 Q777 KV5003 137 / 144 us; but B1 H16 S4096 493 / 417 us: both passes slow down while
  // they share the chip.
  p.overlap = kv_items < sms ? 1 : 0;

  const long long rows = static_cast<long long>(q_heads) * p.nq * kTile;
  const long long blocks = rows / 16;
  if (blocks > INT_MAX) return AVO_B200_EINVAL;
  if (!host::launch_early(bwd::stats_kernel, static_cast<unsigned>(blocks), 256u, 0, st,
                          static_cast<const uint4*>(dout), static_cast<const uint4*>(out), lse,
                          static_cast<float*>(workspace), rows, seq_q, p.nq))
    return AVO_B200_ELAUNCH;
  p.g1 = dk;
  p.g2 = dv;
  if (!host::launch_early(bwd::attn_bwd_kernel<false>, static_cast<unsigned>(kv_items < sms ? kv_items : sms),
                          bwd::kBwdThreads, bwd::kBwdSmemBytes, st, tk, tv, tq, tdo, p))
    return AVO_B200_ELAUNCH;
  p.g1 = dq;
  p.g2 = nullptr;
  p.x1 = q;
  if (!host::launch_early(bwd::attn_bwd_kernel<true>, static_cast<unsigned>(q_items < sms ? q_items : sms),
                          bwd::kBwdThreads, bwd::kBwdSmemBytes, st, tq, tdo, tk, tv, p))
    return AVO_B200_ELAUNCH;
  return cudaGetLastError() == cudaSuccess ? AVO_B200_OK : AVO_B200_ELAUNCH;
}
