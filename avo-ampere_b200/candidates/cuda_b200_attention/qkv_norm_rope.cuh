// From a fused projection to attention's inputs in one pass, and its gradient (B200).
//
// The projection holds, per token, H query heads, G key heads and G value heads of 128
// values.  Query and key heads are normed, x_hat = x * r with r = (mean x^2 + eps)^-1/2,
// weighted, and the first `rot` values rotated by position: a pair (a, b) of column f turns
// to (a cos - b sin, b cos + a sin), cos and sin from a table row per position (one position
// per token, or one per axis, each axis owning a run of columns).  Every head is written to
// its place in [batch, head, token, 128], the layout attention reads; value heads only move.
//
// With p the value a pair's other half holds and sigma = -1 for a, +1 for b:
//     y = r * (x * (w cos) + p * (sigma w_p sin))
// so the norm weight and the rotation fold into two coefficients per column and token, kept
// in registers over all heads of a token.  The gradient turns dy back (g = dy cos - sigma
// p(dy) sin) and passes the norm: dw = sum g x_hat, dx = r (g w - x_hat mean(g w x_hat)); r
// is recomputed from x, nothing is saved.
//
// Both directions move bytes: 16 lanes hold one head's row (8 values a lane, both halves of its
// pairs among them, so a rotation needs no other lane), a half-warp owns one token and walks
// `heads_per_task` of its heads, four rows in flight at a time.  Everything is fp32 between
// the load and one rounding to bf16.  The weights' gradients are summed per thread, then per
// CTA, then over CTAs by a second kernel, each in a fixed order: equal inputs give equal bits.
//
// Memory bandwidth bounds both.  Measured on B200, B4 S4096 H16 Hkv4 (inputs not in L2), calls
// back to back / among other work: the forward 33.8 / 35.1 us (5.8 TB/s) against 31 at the rate
// of a plain copy; the gradient 56.5 / 59.2 us (4.9 TB/s) against 44.  The gradient's issue slots are 60 % busy with a quarter of the warps
// resident (its registers), so computing and fetching do not overlap fully.
#pragma once

#include <cuda_bf16.h>

#include "sm100_ptx.cuh"

namespace avo_b200 {
namespace rope {

constexpr int kRow = 128;
constexpr int kThreadsRope = 128;
constexpr int kWarps = kThreadsRope / 32;
constexpr int kMaxAxes = 4;
constexpr int kUnroll = 4;              // rows in flight per half-warp
constexpr int kFwdCtasPerSm = 8;        // resident CTAs (bounds the registers)
constexpr int kBwdCtasPerSm = 4;
constexpr int kStatusPosition = 4;      // a position lies outside the table

struct RopeParams {
  const __nv_bfloat16* qkv;
  long long stride_b, stride_s;         // elements between batches and tokens of qkv
  __nv_bfloat16* q;                     // outputs (forward) or incoming gradients (backward)
  __nv_bfloat16* k;
  __nv_bfloat16* v;
  __nv_bfloat16* dqkv;                  // backward: [batch, seq, H + 2 G, 128]
  float* partial;                       // backward: [CTAs][2][128] weight gradient sums
  const void* q_weight;                 // null: no norm
  const void* k_weight;
  int weight_bf16;
  const float* cos;                     // [table_rows, rot / 2]
  const float* sin;
  int table_rows;
  const void* pos;                      // null: position = token index
  int pos64;
  long long pos_sa, pos_sb, pos_ss;     // elements between axes, batches, tokens
  int axes;
  int end[kMaxAxes];                    // first column past each axis
  int seq, heads, kv_heads, rot;
  int tokens;                           // batch * seq
  float eps;
  int* status;
  int heads_per_task;
  int segs_q, segs_kv;                  // tasks per token pair: query heads, key (or value) heads
  uint32_t q_tasks, k_tasks, tasks;     // query tasks, then key tasks, then value tasks
  // ceil(2^64 / x) of segs_q, segs_kv and seq (see div_by)
  unsigned long long segs_q_magic, segs_kv_magic, seq_magic;
};

// w / div for every 32-bit w: the high half of w * ceil(2^64 / div).
__device__ __forceinline__ uint32_t div_by(uint32_t w, uint32_t div, unsigned long long magic) {
  return div == 1 ? w : static_cast<uint32_t>(__umul64hi(w, magic));
}

__device__ __forceinline__ float lo_f(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_f(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// The 8 columns of lane l: two groups of 4.  Pairs (f, f + rot/2): 4 first halves and their 4
// second halves.  Interleaved pairs, and columns past the rotated part: 8 in a row.
struct Columns {
  int lo, hi;
  bool turned;
};
template <bool kInterleaved>
__device__ __forceinline__ Columns columns_of(int l, int rot) {
  const bool turned = l * 8 < rot;
  if (kInterleaved || !turned) return {l * 8, l * 8 + 4, turned};
  return {l * 4, (rot >> 1) + l * 4, true};
}

// A row's 8 values of this lane as four bf16 pairs.
template <bool kInterleaved>
__device__ __forceinline__ uint4 load_row(const __nv_bfloat16* row, const Columns& c) {
  if (kInterleaved) return __ldg(reinterpret_cast<const uint4*>(row + c.lo));
  const uint2 a = __ldg(reinterpret_cast<const uint2*>(row + c.lo));
  const uint2 b = __ldg(reinterpret_cast<const uint2*>(row + c.hi));
  return make_uint4(a.x, a.y, b.x, b.y);
}

// The same on its way to 16 bytes of shared memory.
template <bool kInterleaved>
__device__ __forceinline__ void fetch_row(uint32_t to, const __nv_bfloat16* row, const Columns& c) {
  if (kInterleaved) {
    copy_async<16>(to, row + c.lo);
  } else {
    copy_async<8>(to, row + c.lo);
    copy_async<8>(to + 8, row + c.hi);
  }
}

template <bool kInterleaved>
__device__ __forceinline__ void store_row(__nv_bfloat16* row, const Columns& c, uint4 v) {
  if (kInterleaved) {
    *reinterpret_cast<uint4*>(row + c.lo) = v;
  } else {
    *reinterpret_cast<uint2*>(row + c.lo) = make_uint2(v.x, v.y);
    *reinterpret_cast<uint2*>(row + c.hi) = make_uint2(v.z, v.w);
  }
}

// Four values of a weight from column `col` (a multiple of 4).
__device__ __forceinline__ void load_weight4(const void* w, int bf16, int col, float* out) {
  if (bf16) {
    const uint2 a = __ldg(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(w) + col));
    out[0] = lo_f(a.x);
    out[1] = hi_f(a.x);
    out[2] = lo_f(a.y);
    out[3] = hi_f(a.y);
  } else {
    const float4 a = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(w) + col));
    out[0] = a.x;
    out[1] = a.y;
    out[2] = a.z;
    out[3] = a.w;
  }
}

__device__ __forceinline__ void load_weights(const void* w, int bf16, const Columns& c, float (&out)[8]) {
  load_weight4(w, bf16, c.lo, out);
  load_weight4(w, bf16, c.hi, out + 4);
}

// One task: a pair of tokens (one per half-warp) and a run of their heads of one kind.  All
// query tasks come first, then the key tasks, then the value tasks, so that the warps of a CTA
// have equal work and a warp that walks many tasks changes kind twice at most.
struct Task {
  int kind;       // 0 query, 1 key, 2 value
  int h0, h1;     // heads of that kind
  int token;      // this half-warp's token
  bool valid;
  int batch, s;
};

__device__ __forceinline__ Task decode(const RopeParams& p, uint32_t task, int half) {
  Task t;
  t.kind = task < p.q_tasks ? 0 : (task < p.q_tasks + p.k_tasks ? 1 : 2);
  task -= t.kind == 0 ? 0 : (t.kind == 1 ? p.q_tasks : p.q_tasks + p.k_tasks);
  const uint32_t segs = t.kind == 0 ? p.segs_q : p.segs_kv;
  const uint32_t pair = div_by(task, segs, t.kind == 0 ? p.segs_q_magic : p.segs_kv_magic);
  t.h0 = static_cast<int>(task - pair * segs) * p.heads_per_task;
  t.h1 = min(t.kind == 0 ? p.heads : p.kv_heads, t.h0 + p.heads_per_task);
  const uint32_t token = 2 * pair + half;
  t.valid = token < static_cast<uint32_t>(p.tokens);
  t.token = t.valid ? static_cast<int>(token) : p.tokens - 1;
  t.batch = static_cast<int>(div_by(t.token, p.seq, p.seq_magic));
  t.s = t.token - t.batch * p.seq;
  return t;
}

// First head of a kind in the projection, and its place in [batch, heads, seq, 128].
__device__ __forceinline__ int first_head(const RopeParams& p, int kind) {
  return kind == 0 ? 0 : (kind == 1 ? p.heads : p.heads + p.kv_heads);
}
__device__ __forceinline__ long long row_at(const RopeParams& p, const Task& t, int h) {
  return ((static_cast<long long>(t.batch) * (t.kind == 0 ? p.heads : p.kv_heads) + h) * p.seq + t.s) * kRow;
}

// The table rows of a token, one per axis; whether one of them lies outside (then row 0).  The
// position of an axis that owns no columns is not looked at: nothing is read for it.
struct TableRows {
  long long row[kMaxAxes];
  bool bad;
};
__device__ __forceinline__ TableRows table_rows(const RopeParams& p, const Task& t) {
  TableRows rows;
  rows.bad = false;
#pragma unroll
  for (int a = 0; a < kMaxAxes; ++a) {
    rows.row[a] = 0;
    if (a < p.axes && p.end[a] > (a > 0 ? p.end[a - 1] : 0)) {
      long long r = t.s;
      if (p.pos != nullptr) {
        const long long at = a * p.pos_sa + t.batch * p.pos_sb + t.s * p.pos_ss;
        r = p.pos64 ? __ldg(static_cast<const long long*>(p.pos) + at) : __ldg(static_cast<const int*>(p.pos) + at);
      }
      if (r < 0 || r >= p.table_rows) {
        rows.bad = true;
        r = 0;
      }
      rows.row[a] = r;
    }
  }
  return rows;
}

// Where table column f of a token lies.
__device__ __forceinline__ long long table_at(const RopeParams& p, const TableRows& rows, int f) {
  long long r = rows.row[0];
#pragma unroll
  for (int a = 1; a < kMaxAxes; ++a)
    if (a < p.axes && f >= p.end[a - 1]) r = rows.row[a];
  return r * (p.rot >> 1) + f;
}

// cos and sigma * sin of this lane's 8 columns (1 and 0 past the rotated part), from those of
// the 4 pairs that it turns.
template <bool kInterleaved>
__device__ __forceinline__ void spread_turn(bool turned, bool bad, const float4& cc4, const float4& ss4, float (&c)[8],
                                            float (&s)[8]) {
  const float nan = __int_as_float(0x7fc00000);
  const float cc[4] = {cc4.x, cc4.y, cc4.z, cc4.w}, ss[4] = {ss4.x, ss4.y, ss4.z, ss4.w};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int i = kInterleaved ? e >> 1 : e & 3;
    const bool minus = kInterleaved ? (e & 1) == 0 : e < 4;
    c[e] = !turned ? 1.f : bad ? nan : cc[i];
    s[e] = !turned ? 0.f : bad ? nan : (minus ? -ss[i] : ss[i]);
  }
}

template <bool kInterleaved>
__device__ __forceinline__ void load_turn(const RopeParams& p, const Task& t, int l, float (&c)[8], float (&s)[8]) {
  float4 cc = make_float4(1.f, 1.f, 1.f, 1.f), ss = make_float4(0.f, 0.f, 0.f, 0.f);
  bool bad = false;
  const bool turned = l * 8 < p.rot;
  if (turned) {
    const TableRows rows = table_rows(p, t);
    bad = rows.bad;
    if (bad && t.valid && l == 0 && p.status != nullptr) atomicOr(p.status, kStatusPosition);
    const int col = l * 4;  // this lane turns pairs col .. col + 3, table columns of the same index
    if (p.axes == 1) {
      const long long at = table_at(p, rows, col);
      cc = __ldg(reinterpret_cast<const float4*>(p.cos + at));
      ss = __ldg(reinterpret_cast<const float4*>(p.sin + at));
    } else {
      float* const c4 = &cc.x;
      float* const s4 = &ss.x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long long at = table_at(p, rows, col + i);
        c4[i] = __ldg(p.cos + at);
        s4[i] = __ldg(p.sin + at);
      }
    }
  }
  spread_turn<kInterleaved>(turned, bad, cc, ss, c, s);
}

// The same on their way to shared memory (nothing for lanes past the rotated part).
__device__ __forceinline__ bool fetch_turn(const RopeParams& p, const Task& t, int l, uint32_t cos_to, uint32_t sin_to) {
  if (l * 8 >= p.rot) return false;
  const TableRows rows = table_rows(p, t);
  if (rows.bad && t.valid && l == 0 && p.status != nullptr) atomicOr(p.status, kStatusPosition);
  const int col = l * 4;
  if (p.axes == 1) {
    const long long at = table_at(p, rows, col);
    copy_async<16>(cos_to, p.cos + at);
    copy_async<16>(sin_to, p.sin + at);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long at = table_at(p, rows, col + i);
      copy_async<4>(cos_to + 4 * i, p.cos + at);
      copy_async<4>(sin_to + 4 * i, p.sin + at);
    }
  }
  return rows.bad;
}

// Index of the other half of value e of a lane.
template <bool kInterleaved>
__device__ __forceinline__ constexpr int other(int e) {
  return kInterleaved ? e ^ 1 : e ^ 4;
}

__device__ __forceinline__ float half_sum(float v) {
#pragma unroll
  for (int m = 8; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}

// The four packed fp32 pairs of a lane's values, and the pairs of their other halves.
__device__ __forceinline__ void unpack4(uint4 x, uint64_t (&f)[4]) {
  f[0] = f2_pack(lo_f(x.x), hi_f(x.x));
  f[1] = f2_pack(lo_f(x.y), hi_f(x.y));
  f[2] = f2_pack(lo_f(x.z), hi_f(x.z));
  f[3] = f2_pack(lo_f(x.w), hi_f(x.w));
}
template <bool kInterleaved>
__device__ __forceinline__ void others4(uint4 x, const uint64_t (&f)[4], uint64_t (&g)[4]) {
  if (kInterleaved) {
    g[0] = f2_pack(hi_f(x.x), lo_f(x.x));
    g[1] = f2_pack(hi_f(x.y), lo_f(x.y));
    g[2] = f2_pack(hi_f(x.z), lo_f(x.z));
    g[3] = f2_pack(hi_f(x.w), lo_f(x.w));
  } else {
    g[0] = f[2];
    g[1] = f[3];
    g[2] = f[0];
    g[3] = f[1];
  }
}

__device__ __forceinline__ uint4 pack4(const uint64_t (&f)[4]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b;
    f2_unpack(f[i], a, b);
    w[i] = pack_bf16x2(a, b);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ float sum2(const uint64_t v) {
  float a, b;
  f2_unpack(v, a, b);
  return a + b;
}

// Sum over the row of u * v (packed pairs).
__device__ __forceinline__ float row_dot(const uint64_t (&u)[4], const uint64_t (&v)[4]) {
  uint64_t a = f2_mul(u[0], v[0]), b = f2_mul(u[1], v[1]);
  a = f2_fma(u[2], v[2], a);
  b = f2_fma(u[3], v[3], b);
  return half_sum(sum2(f2_add(a, b)));
}

template <bool kInterleaved>
__global__ void __launch_bounds__(kThreadsRope, kFwdCtasPerSm)
    qkv_norm_rope_kernel(const __grid_constant__ RopeParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x & 31, l = lane & 15, half = lane >> 4;
  const uint32_t task = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (task >= p.tasks) return;
  const Task t = decode(p, task, half);
  const Columns col = columns_of<kInterleaved>(l, p.rot);
  const __nv_bfloat16* src =
      p.qkv + t.batch * p.stride_b + t.s * p.stride_s + static_cast<long long>(first_head(p, t.kind) + t.h0) * kRow;
  const long long step = static_cast<long long>(p.seq) * kRow;
  __nv_bfloat16* dst = (t.kind == 0 ? p.q : (t.kind == 1 ? p.k : p.v)) + row_at(p, t, t.h0);
  // Rows past the run compute on ones and are not stored: without branches the rows' sums
  // (shuffles) overlap.
  const uint4 ones = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);
  uint4 x[kUnroll];
  int left = t.h1 - t.h0;
  auto load = [&]() {
#pragma unroll
    for (int i = 0; i < kUnroll; ++i)
      x[i] = i < left ? load_row<kInterleaved>(src + i * kRow, col) : ones;
    src += kUnroll * kRow;
  };
  load();
  if (t.kind == 2) {
    for (; left > 0; left -= kUnroll, dst += kUnroll * step) {
      if (left < t.h1 - t.h0) load();
#pragma unroll
      for (int i = 0; i < kUnroll; ++i)
        if (i < left && t.valid) store_row<kInterleaved>(dst + i * step, col, x[i]);
    }
    return;
  }
  const bool norm = p.q_weight != nullptr;
  uint64_t a[4], b[4];
  {
    float c[8], s[8];
    load_turn<kInterleaved>(p, t, l, c, s);
    if (norm) {
      float w[8];
      load_weights(t.kind == 0 ? p.q_weight : p.k_weight, p.weight_bf16, col, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        c[e] *= w[e];
        s[e] *= col.turned ? w[other<kInterleaved>(e)] : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = f2_pack(c[2 * i], c[2 * i + 1]);
      b[i] = f2_pack(s[2 * i], s[2 * i + 1]);
    }
  }
  for (; left > 0; left -= kUnroll, dst += kUnroll * step) {
    if (left < t.h1 - t.h0) load();
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      uint64_t f[4], g[4];
      unpack4(x[i], f);
      others4<kInterleaved>(x[i], f, g);
      const float r = norm ? rsqrtf(row_dot(f, f) * (1.f / kRow) + p.eps) : 1.f;
      const uint64_t r2 = f2_pack(r, r);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = f2_mul(r2, f2_fma(g[e], b[e], f2_mul(f[e], a[e])));
      if (i < left && t.valid) store_row<kInterleaved>(dst + i * step, col, pack4(f));
    }
  }
}

// Groups of kUnroll rows go through shared memory: while a group is computed, the next one of
// the warp (and the table rows, at a task's start) is on its way.  Every thread reads only what
// it has fetched itself, so no barrier is needed.  (Measured as above: without this 64.2 us,
// registers being full; with it 58.7; with 5 CTAs of 2, 3 or 4 rows a group 62.4, 69.4, 75.0.)
template <bool kInterleaved>
__global__ void __launch_bounds__(kThreadsRope, kBwdCtasPerSm)
    qkv_norm_rope_bwd_kernel(const __grid_constant__ RopeParams p) {
  __shared__ float sums[kWarps][2][kRow];
  __shared__ uint4 ring[2][2 * kUnroll][kThreadsRope];  // dy rows, then x rows, of a group
  __shared__ float4 turns[2][2][kThreadsRope];
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x & 31, l = lane & 15, half = lane >> 4, warp = threadIdx.x >> 5;
  const bool norm = p.q_weight != nullptr;
  const Columns col = columns_of<kInterleaved>(l, p.rot);
  const long long step = static_cast<long long>(p.seq) * kRow;
  uint64_t dw[4];  // weight gradient of the current kind
  auto clear = [&]() {
#pragma unroll
    for (int e = 0; e < 4; ++e) dw[e] = f2_pack(0.f, 0.f);
  };
  // Adds the two half-warps and leaves the warp's sum of `kind` in shared memory.
  auto flush = [&](int kind) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float v0, v1;
      f2_unpack(dw[e >> 1], v0, v1);
      float v = e & 1 ? v1 : v0;
      v += __shfl_xor_sync(0xffffffffu, v, 16);
      if (half == 0) sums[warp][kind][(e < 4 ? col.lo : col.hi) + (e & 3)] = v;
    }
    clear();
  };
  clear();
  int kind = 0;

  // The group that is fetched: its task's place, and how many of the task's rows are left.
  unsigned long long task = blockIdx.x * kWarps + warp;
  const __nv_bfloat16 *in = nullptr, *src = nullptr;
  __nv_bfloat16* dst = nullptr;
  int left = 0, next_kind = 0, tasks_begun = 0;
  bool first = false, valid = false, bad = false;
  auto begin_task = [&]() {
    const Task t = decode(p, static_cast<uint32_t>(task), half);
    const int h_at = first_head(p, t.kind) + t.h0;
    src = p.qkv + t.batch * p.stride_b + t.s * p.stride_s + static_cast<long long>(h_at) * kRow;
    dst = p.dqkv + (static_cast<long long>(t.token) * (p.heads + 2 * p.kv_heads) + h_at) * kRow;
    in = (t.kind == 0 ? p.q : (t.kind == 1 ? p.k : p.v)) + row_at(p, t, t.h0);
    left = t.h1 - t.h0;
    next_kind = t.kind;
    valid = t.valid;
    first = true;
    ++tasks_begun;
    if (t.kind < 2) {
      float4* const to = &turns[tasks_begun & 1][0][threadIdx.x];
      bad = fetch_turn(p, t, l, smem_addr(to), smem_addr(to + kThreadsRope));
    }
  };
  auto fetch = [&](int stage) {
    const uint32_t to = smem_addr(&ring[stage][0][threadIdx.x]);
    constexpr uint32_t kNext = kThreadsRope * sizeof(uint4);
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      if (i >= left) break;
      fetch_row<kInterleaved>(to + i * kNext, in + i * step, col);
      if (next_kind < 2 && norm) fetch_row<kInterleaved>(to + (kUnroll + i) * kNext, src + i * kRow, col);
    }
  };
  const uint4 ones = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);
  uint64_t c2[4], s2[4], w2[4];
  bool more = task < p.tasks;
  if (more) {
    begin_task();
    fetch(0);
  }
  copy_async_commit();
  for (int stage = 0; more; stage ^= 1) {
    // This group; then the next one is fetched.
    __nv_bfloat16* const out = dst;
    const int rows = valid ? left : 0, this_kind = next_kind, turn = tasks_begun & 1;
    const bool begun = first, nan = bad;
    first = false;
    left -= kUnroll;
    in += kUnroll * step;
    src += kUnroll * kRow;
    dst += kUnroll * kRow;
    if (left <= 0) {
      task += gridDim.x * kWarps;
      more = task < p.tasks;
      if (more) begin_task();
    }
    if (more) fetch(stage ^ 1);
    copy_async_commit();
    copy_async_wait<1>();
    const uint4* const from = &ring[stage][0][threadIdx.x];
    if (this_kind == 2) {
#pragma unroll
      for (int i = 0; i < kUnroll; ++i)
        if (i < rows) store_row<kInterleaved>(out + i * kRow, col, from[i * kThreadsRope]);
      continue;
    }
    if (begun) {
      for (; kind < this_kind; ++kind)
        if (norm) flush(kind);
      float c[8], s[8], w[8];
      const float4* const at = &turns[turn][0][threadIdx.x];
      spread_turn<kInterleaved>(col.turned, nan, at[0], at[kThreadsRope], c, s);
      if (norm) load_weights(this_kind == 0 ? p.q_weight : p.k_weight, p.weight_bf16, col, w);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        c2[i] = f2_pack(c[2 * i], c[2 * i + 1]);
        s2[i] = f2_pack(-s[2 * i], -s[2 * i + 1]);
        w2[i] = norm ? f2_pack(w[2 * i], w[2 * i + 1]) : 0;
      }
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      // (Rows past the run, or of the token past the last: a zero gradient on ones.)
      const uint4 d = i < rows ? from[i * kThreadsRope] : make_uint4(0u, 0u, 0u, 0u);
      uint64_t g[4], o[4], turned[4];
      unpack4(d, g);
      others4<kInterleaved>(d, g, o);
#pragma unroll
      for (int e = 0; e < 4; ++e) turned[e] = f2_fma(o[e], s2[e], f2_mul(g[e], c2[e]));
      if (norm) {
        const uint4 x = i < rows ? from[(kUnroll + i) * kThreadsRope] : ones;
        uint64_t f[4], gw[4];
        unpack4(x, f);
        // The two sums of the row are taken side by side: mean(g w x_hat) = r mean(g w x).
#pragma unroll
        for (int e = 0; e < 4; ++e) gw[e] = f2_mul(turned[e], w2[e]);
        const float sq = row_dot(f, f), dot = row_dot(gw, f);
        const float r = rsqrtf(sq * (1.f / kRow) + p.eps);
        const float m = -dot * (1.f / kRow) * r;
        const uint64_t r2 = f2_pack(r, r), m2 = f2_pack(m, m);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f[e] = f2_mul(f[e], r2);  // x_hat
          dw[e] = f2_fma(turned[e], f[e], dw[e]);
          turned[e] = f2_mul(r2, f2_fma(f[e], m2, gw[e]));
        }
      }
      if (i < rows) store_row<kInterleaved>(out + i * kRow, col, pack4(turned));
    }
  }
  copy_async_wait<0>();
  if (!norm) return;
  for (; kind < 2; ++kind) flush(kind);
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * kRow; i += kThreadsRope) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) v += (&sums[k][0][0])[i];
    p.partial[static_cast<long long>(blockIdx.x) * (2 * kRow) + i] = v;
  }
}

// dw[col] = sum over CTAs of partial[cta][col]: 8 columns (a sector of memory) per block, 128
// threads per column, so that a thread has only a few rows, all in flight at once (measured on
// B200, B4 S4096 H16 Hkv4, the whole gradient: 57.0 us with 32 columns per block, 56.7 with 8).
constexpr int kSumCols = 8;
__global__ void __launch_bounds__(1024)
    weight_grad_kernel(const float* __restrict__ partial, int ctas, float* __restrict__ dq_weight,
                       float* __restrict__ dk_weight) {
  constexpr int kRows = 1024 / kSumCols;
  __shared__ float sums[32][kSumCols];
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = lane % kSumCols, col = blockIdx.x * kSumCols + c;
  const float* from = partial + col;
  float v = 0.f;
#pragma unroll 8
  for (int row = threadIdx.x / kSumCols; row < ctas; row += kRows) v += __ldcg(from + row * (2 * kRow));
  // The four rows of a warp, then the 32 warps.
  v += __shfl_xor_sync(0xffffffffu, v, 8);
  v += __shfl_xor_sync(0xffffffffu, v, 16);
  if (lane < kSumCols) sums[warp][lane] = v;
  __syncthreads();
  if (warp == 0) {
    float total = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) total += sums[(lane / kSumCols) * 8 + k][c];
    total += __shfl_xor_sync(0xffffffffu, total, 8);
    total += __shfl_xor_sync(0xffffffffu, total, 16);
    if (lane < kSumCols) {
      if (col < kRow)
        dq_weight[col] = total;
      else
        dk_weight[col - kRow] = total;
    }
  }
}

}  // namespace rope
}  // namespace avo_b200
