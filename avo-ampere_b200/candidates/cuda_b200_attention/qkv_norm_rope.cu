// C-ABI entry points of the QKV norm + rotation (declared in include/avo_b200_attn.h).
#include <climits>
#include <cmath>

#include "avo_b200_attn.h"
#include "host_common.h"
#include "qkv_norm_rope.cuh"

namespace avo_b200 {
namespace {

// What both directions share: checks and fills everything but the in/out tensors.
int fill(rope::RopeParams& p, const void* qkv, long long stride_b, long long stride_s, int batch, int seq, int heads,
         int kv_heads, int head_dim, const void* q_weight, const void* k_weight, int weight_bf16, const float* cos,
         const float* sin, int table_rows, int rotary_dim, const void* positions, int positions_int64,
         long long pos_sa, long long pos_sb, long long pos_ss, int axes, const int* sections, float eps, int* status) {
  if (head_dim != rope::kRow || batch < 0 || seq < 0 || heads < 0 || kv_heads < 0) return AVO_B200_EINVAL;
  if (rotary_dim <= 0 || rotary_dim > rope::kRow || rotary_dim % 16 != 0) return AVO_B200_EINVAL;
  if (axes < 1 || axes > rope::kMaxAxes || (axes > 1 && (sections == nullptr || positions == nullptr)))
    return AVO_B200_EINVAL;
  if ((q_weight == nullptr) != (k_weight == nullptr) || !(eps >= 0.f) || !std::isfinite(eps)) return AVO_B200_EINVAL;
  const long long tokens = static_cast<long long>(batch) * seq;
  const long long all = static_cast<long long>(heads) + 2ll * kv_heads;
  if (tokens > INT_MAX || all > INT_MAX / rope::kRow) return AVO_B200_EINVAL;
  p.tokens = static_cast<int>(tokens);
  if (tokens == 0 || all == 0) return AVO_B200_OK;
  if (qkv == nullptr || !host::aligned(qkv, 16) || stride_b % 8 != 0 || stride_s % 8 != 0) return AVO_B200_EINVAL;
  if (cos == nullptr || sin == nullptr || !host::aligned(cos, 16) || !host::aligned(sin, 16) || table_rows < 1)
    return AVO_B200_EINVAL;
  if (positions == nullptr && seq > table_rows) return AVO_B200_EINVAL;
  if (positions != nullptr && !host::aligned(positions, positions_int64 ? 8 : 4)) return AVO_B200_EINVAL;
  if (q_weight != nullptr && (!host::aligned(q_weight, 16) || !host::aligned(k_weight, 16))) return AVO_B200_EINVAL;
  p.qkv = static_cast<const __nv_bfloat16*>(qkv);
  p.stride_b = stride_b;
  p.stride_s = stride_s;
  p.q_weight = q_weight;
  p.k_weight = k_weight;
  p.weight_bf16 = weight_bf16 != 0;
  p.cos = cos;
  p.sin = sin;
  p.table_rows = table_rows;
  p.pos = positions;
  p.pos64 = positions_int64 != 0;
  p.pos_sa = pos_sa;
  p.pos_sb = pos_sb;
  p.pos_ss = pos_ss;
  p.axes = axes;
  int end = 0;
  for (int a = 0; a < rope::kMaxAxes; ++a) {
    if (a < axes) {
      const int n = axes == 1 ? rotary_dim / 2 : sections[a];
      if (n < 0 || n > rotary_dim / 2) return AVO_B200_EINVAL;
      end += n;
    }
    p.end[a] = end;
  }
  if (end != rotary_dim / 2) return AVO_B200_EINVAL;
  p.seq = seq;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.rot = rotary_dim;
  p.eps = eps;
  p.status = status;
  return AVO_B200_OK;
}

// Heads per task: a task reads its token's table rows once and a contiguous run of memory, so
// that more heads share them, but there have to be enough tasks (warps) to keep every
// multiprocessor's memory queue full.  (Measured on B200, B4 S4096 H16 Hkv4, up to 16 / 12 / 8 / 4
// heads: forward 35.0 / 37.4 / 35.7 / 39.9 us, gradient 56.8 / 64.3 / 59.8 / 64.3.)  False where
// the tasks cannot be counted in 31 bits.
bool split_heads(rope::RopeParams& p, int sms) {
  const long long pairs = (static_cast<long long>(p.tokens) + 1) / 2;
  auto segs = [](int heads, int per) { return (heads + per - 1) / per; };
  int per = 16;
  while (per > 1 && pairs * (segs(p.heads, per) + 2 * segs(p.kv_heads, per)) < 64ll * sms) per /= 2;
  p.heads_per_task = per;
  p.segs_q = segs(p.heads, per);
  p.segs_kv = segs(p.kv_heads, per);
  const long long q_tasks = pairs * p.segs_q, k_tasks = pairs * p.segs_kv;
  if (q_tasks + 2 * k_tasks > INT_MAX) return false;  // (about 10^13 bytes)
  p.q_tasks = static_cast<uint32_t>(q_tasks);
  p.k_tasks = static_cast<uint32_t>(k_tasks);
  p.tasks = p.q_tasks + 2 * p.k_tasks;
  auto magic = [](int x) { return x > 0 ? ~0ull / static_cast<unsigned>(x) + 1 : 0; };  // unused for 1
  p.segs_q_magic = magic(p.segs_q);
  p.segs_kv_magic = magic(p.segs_kv);
  p.seq_magic = magic(p.seq);
  return true;
}

long long ctas_for(long long tasks) { return (tasks + rope::kWarps - 1) / rope::kWarps; }

bool all_aligned(const void* a, const void* b, const void* c) {
  return host::aligned(a, 16) && host::aligned(b, 16) && host::aligned(c, 16);
}

}  // namespace
}  // namespace avo_b200

using namespace avo_b200;

extern "C" int avo_b200_qkv_norm_rope(const void* qkv, long long batch_stride, long long token_stride, void* q, void* k,
                                      void* v, int batch, int seq, int heads, int kv_heads, int head_dim,
                                      const void* q_weight, const void* k_weight, int weight_bf16, const float* cos,
                                      const float* sin, int table_rows, int rotary_dim, int interleaved,
                                      const void* positions, int positions_int64, long long pos_axis_stride,
                                      long long pos_batch_stride, long long pos_token_stride, int axes,
                                      const int* sections, float eps, int* status_dev, void* stream) {
  rope::RopeParams p{};
  int rc = fill(p, qkv, batch_stride, token_stride, batch, seq, heads, kv_heads, head_dim, q_weight, k_weight,
                weight_bf16, cos, sin, table_rows, rotary_dim, positions, positions_int64, pos_axis_stride,
                pos_batch_stride, pos_token_stride, axes, sections, eps, status_dev);
  if (rc != AVO_B200_OK) return rc;
  if (p.tokens == 0 || heads + kv_heads == 0) return AVO_B200_OK;
  if ((heads > 0 && q == nullptr) || (kv_heads > 0 && (k == nullptr || v == nullptr)) || !all_aligned(q, k, v))
    return AVO_B200_EINVAL;
  int sms = 0;
  if ((rc = host::device(&sms)) != AVO_B200_OK) return rc;
  p.q = static_cast<__nv_bfloat16*>(q);
  p.k = static_cast<__nv_bfloat16*>(k);
  p.v = static_cast<__nv_bfloat16*>(v);
  if (!split_heads(p, sms)) return AVO_B200_EINVAL;
  const long long ctas = ctas_for(p.tasks);
  auto* kernel = interleaved ? rope::qkv_norm_rope_kernel<true> : rope::qkv_norm_rope_kernel<false>;
  if (!host::launch_early(kernel, static_cast<unsigned>(ctas), rope::kThreadsRope, 0,
                          static_cast<cudaStream_t>(stream), p))
    return AVO_B200_ELAUNCH;
  return cudaGetLastError() == cudaSuccess ? AVO_B200_OK : AVO_B200_ELAUNCH;
}

extern "C" int avo_b200_qkv_norm_rope_bwd_workspace_size(size_t* bytes) {
  if (bytes == nullptr) return AVO_B200_EINVAL;
  int sms = 0;
  const int rc = host::device(&sms);
  if (rc != AVO_B200_OK) return rc;
  *bytes = static_cast<size_t>(sms) * rope::kBwdCtasPerSm * 2 * rope::kRow * sizeof(float);
  return AVO_B200_OK;
}

extern "C" int avo_b200_qkv_norm_rope_bwd(const void* dq, const void* dk, const void* dv, const void* qkv,
                                          long long batch_stride, long long token_stride, void* dqkv,
                                          float* dq_weight, float* dk_weight, int batch, int seq, int heads,
                                          int kv_heads, int head_dim, const void* q_weight, const void* k_weight,
                                          int weight_bf16, const float* cos, const float* sin, int table_rows,
                                          int rotary_dim, int interleaved, const void* positions,
                                          int positions_int64, long long pos_axis_stride, long long pos_batch_stride,
                                          long long pos_token_stride, int axes, const int* sections, float eps,
                                          void* workspace, size_t workspace_bytes, int* status_dev, void* stream) {
  rope::RopeParams p{};
  int rc = fill(p, qkv, batch_stride, token_stride, batch, seq, heads, kv_heads, head_dim, q_weight, k_weight,
                weight_bf16, cos, sin, table_rows, rotary_dim, positions, positions_int64, pos_axis_stride,
                pos_batch_stride, pos_token_stride, axes, sections, eps, status_dev);
  if (rc != AVO_B200_OK) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool norm = q_weight != nullptr;
  if (norm && (dq_weight == nullptr || dk_weight == nullptr || !host::aligned(dq_weight, 4) ||
               !host::aligned(dk_weight, 4)))
    return AVO_B200_EINVAL;
  if (p.tokens == 0 || heads + kv_heads == 0) {
    if (norm && (cudaMemsetAsync(dq_weight, 0, rope::kRow * sizeof(float), st) != cudaSuccess ||
                 cudaMemsetAsync(dk_weight, 0, rope::kRow * sizeof(float), st) != cudaSuccess)) {
      (void)cudaGetLastError();
      return AVO_B200_ELAUNCH;
    }
    return AVO_B200_OK;
  }
  if ((heads > 0 && dq == nullptr) || (kv_heads > 0 && (dk == nullptr || dv == nullptr)) || !all_aligned(dq, dk, dv))
    return AVO_B200_EINVAL;
  if (dqkv == nullptr || !host::aligned(dqkv, 16)) return AVO_B200_EINVAL;
  int sms = 0;
  if ((rc = host::device(&sms)) != AVO_B200_OK) return rc;
  p.q = static_cast<__nv_bfloat16*>(const_cast<void*>(dq));
  p.k = static_cast<__nv_bfloat16*>(const_cast<void*>(dk));
  p.v = static_cast<__nv_bfloat16*>(const_cast<void*>(dv));
  p.dqkv = static_cast<__nv_bfloat16*>(dqkv);
  if (!split_heads(p, sms)) return AVO_B200_EINVAL;
  long long ctas = ctas_for(p.tasks);
  const long long most = static_cast<long long>(sms) * rope::kBwdCtasPerSm;
  if (ctas > most) ctas = most;
  if (norm && (workspace == nullptr || !host::aligned(workspace, 16) ||
               workspace_bytes < static_cast<size_t>(ctas) * 2 * rope::kRow * sizeof(float)))
    return AVO_B200_EINVAL;
  p.partial = static_cast<float*>(workspace);
  auto* kernel = interleaved ? rope::qkv_norm_rope_bwd_kernel<true> : rope::qkv_norm_rope_bwd_kernel<false>;
  if (!host::launch_early(kernel, static_cast<unsigned>(ctas), rope::kThreadsRope, 0, st, p)) return AVO_B200_ELAUNCH;
  if (norm && !host::launch_early(rope::weight_grad_kernel, 2 * rope::kRow / rope::kSumCols, 1024u, 0, st,
                                  static_cast<const float*>(p.partial), static_cast<int>(ctas), dq_weight, dk_weight))
    return AVO_B200_ELAUNCH;
  return cudaGetLastError() == cudaSuccess ? AVO_B200_OK : AVO_B200_ELAUNCH;
}
