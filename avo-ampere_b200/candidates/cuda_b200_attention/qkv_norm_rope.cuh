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
// Both directions move bytes: 16 lanes hold one head's row (16 bytes a lane, so a row is one
// 256-byte access), a half-warp owns one token and walks `heads_per_task` of its heads, four
// rows in flight at a time.  Everything is fp32 between the load and one rounding to bf16.
// The weights' gradients are summed per thread, then per CTA, then over CTAs by a second
// kernel, each in a fixed order: equal inputs give equal bits.
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
  int segs_q, segs_kv;                  // tasks per token pair: query, key (and value) heads
  long long tasks;
};

__device__ __forceinline__ float lo_f(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_f(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

__device__ __forceinline__ void load_weights(const void* w, int bf16, int col, float (&out)[8]) {
  if (bf16) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(w) + col));
    const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      out[2 * i] = lo_f(u[i]);
      out[2 * i + 1] = hi_f(u[i]);
    }
  } else {
    const float4* f = reinterpret_cast<const float4*>(static_cast<const float*>(w) + col);
    const float4 a = __ldg(f), b = __ldg(f + 1);
    out[0] = a.x; out[1] = a.y; out[2] = a.z; out[3] = a.w;
    out[4] = b.x; out[5] = b.y; out[6] = b.z; out[7] = b.w;
  }
}

// One task: a pair of tokens (one per half-warp) and a run of heads of one kind.
struct Task {
  int kind;       // 0 query, 1 key, 2 value
  int h0, h1;     // heads of that kind
  int token;      // this half-warp's token
  bool valid;
  int batch, s;
};

__device__ __forceinline__ Task decode(const RopeParams& p, long long task, int half) {
  Task t;
  const int per = p.segs_q + 2 * p.segs_kv;
  const long long pair = task / per;
  int seg = static_cast<int>(task - pair * per);
  int heads = p.heads;
  t.kind = 0;
  if (seg >= p.segs_q) {
    seg -= p.segs_q;
    heads = p.kv_heads;
    t.kind = 1;
    if (seg >= p.segs_kv) {
      seg -= p.segs_kv;
      t.kind = 2;
    }
  }
  t.h0 = seg * p.heads_per_task;
  t.h1 = min(heads, t.h0 + p.heads_per_task);
  const long long token = 2 * pair + half;
  t.valid = token < p.tokens;
  t.token = t.valid ? static_cast<int>(token) : p.tokens - 1;
  t.batch = t.token / p.seq;
  t.s = t.token - t.batch * p.seq;
  return t;
}

// cos and sigma * sin of this lane's 8 columns (1 and 0 past the rotated part).
template <bool kInterleaved>
__device__ __forceinline__ void load_turn(const RopeParams& p, const Task& t, int l, float (&c)[8], float (&s)[8]) {
  const int half_lanes = p.rot >> 4;  // lanes per half of the rotated part
  const int half_rot = p.rot >> 1;
  if (l * 8 >= p.rot) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      c[e] = 1.f;
      s[e] = 0.f;
    }
    return;
  }
  long long row[kMaxAxes];
  bool bad = false;
#pragma unroll
  for (int a = 0; a < kMaxAxes; ++a) {
    row[a] = 0;
    if (a < p.axes) {
      long long r = t.s;
      if (p.pos != nullptr) {
        const long long at = a * p.pos_sa + t.batch * p.pos_sb + t.s * p.pos_ss;
        r = p.pos64 ? __ldg(static_cast<const long long*>(p.pos) + at) : __ldg(static_cast<const int*>(p.pos) + at);
      }
      if (r < 0 || r >= p.table_rows) {
        bad = true;
        r = 0;
      }
      row[a] = r;
    }
  }
  if (bad && t.valid && l == 0 && p.status != nullptr) atomicOr(p.status, kStatusPosition);
  constexpr int kCols = kInterleaved ? 4 : 8;  // table columns this lane uses
  const int col = kInterleaved ? l * 4 : (l < half_lanes ? l : l - half_lanes) * 8;
  float cc[kCols], ss[kCols];
  auto row_of = [&](int f) {
    long long r = row[0];
#pragma unroll
    for (int a = 1; a < kMaxAxes; ++a)
      if (a < p.axes && f >= p.end[a - 1]) r = row[a];
    return r;
  };
  const long long first = row_of(col);
  if (p.axes == 1) {
#pragma unroll
    for (int i = 0; i < kCols; i += 4) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(p.cos + first * half_rot + col + i));
      const float4 b = __ldg(reinterpret_cast<const float4*>(p.sin + first * half_rot + col + i));
      cc[i] = a.x; cc[i + 1] = a.y; cc[i + 2] = a.z; cc[i + 3] = a.w;
      ss[i] = b.x; ss[i + 1] = b.y; ss[i + 2] = b.z; ss[i + 3] = b.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kCols; ++i) {
      const long long at = row_of(col + i) * half_rot + col + i;
      cc[i] = __ldg(p.cos + at);
      ss[i] = __ldg(p.sin + at);
    }
  }
  const float nan = __int_as_float(0x7fc00000);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int i = kInterleaved ? e / 2 : e;
    const bool minus = kInterleaved ? (e & 1) == 0 : l < half_lanes;
    c[e] = bad ? nan : cc[i];
    s[e] = bad ? nan : (minus ? -ss[i] : ss[i]);
  }
}

// The other halves of this lane's 8 values (bf16 pairs).  Every lane of the warp calls it.
template <bool kInterleaved>
__device__ __forceinline__ uint4 partner_of(uint4 x, int src_lane) {
  if (kInterleaved) {
    return make_uint4(__funnelshift_l(x.x, x.x, 16), __funnelshift_l(x.y, x.y, 16), __funnelshift_l(x.z, x.z, 16),
                      __funnelshift_l(x.w, x.w, 16));
  }
  return make_uint4(__shfl_sync(0xffffffffu, x.x, src_lane), __shfl_sync(0xffffffffu, x.y, src_lane),
                    __shfl_sync(0xffffffffu, x.z, src_lane), __shfl_sync(0xffffffffu, x.w, src_lane));
}

__device__ __forceinline__ float half_sum(float v) {
#pragma unroll
  for (int m = 8; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}

__device__ __forceinline__ void unpack8(uint4 x, float (&f)[8]) {
  const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = lo_f(u[i]);
    f[2 * i + 1] = hi_f(u[i]);
  }
}

__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}

// Lane of the half-warp that holds the other halves of this lane's columns.
__device__ __forceinline__ int partner_lane(int l, int rot) {
  const int h = rot >> 4;
  return l < h ? l + h : (l < 2 * h ? l - h : l);
}

template <bool kInterleaved>
__global__ void __launch_bounds__(kThreadsRope) qkv_norm_rope_kernel(const __grid_constant__ RopeParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x & 31, l = lane & 15, half = lane >> 4;
  const long long task = static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (task >= p.tasks) return;
  const Task t = decode(p, task, half);
  const int head_base = t.kind == 0 ? 0 : (t.kind == 1 ? p.heads : p.heads + p.kv_heads);
  const int out_heads = t.kind == 0 ? p.heads : p.kv_heads;
  __nv_bfloat16* const dst = t.kind == 0 ? p.q : (t.kind == 1 ? p.k : p.v);
  const __nv_bfloat16* const src = p.qkv + t.batch * p.stride_b + t.s * p.stride_s + l * 8;
  auto out_row = [&](int h) {
    return reinterpret_cast<uint4*>(dst + ((static_cast<long long>(t.batch) * out_heads + h) * p.seq + t.s) * kRow +
                                    l * 8);
  };
  float a[8], b[8];
  const bool norm = p.q_weight != nullptr;
  const int src_lane = half * 16 + partner_lane(l, p.rot);
  if (t.kind < 2) {
    load_turn<kInterleaved>(p, t, l, a, b);
    if (norm) {
      float w[8], wp[8];
      const void* weight = t.kind == 0 ? p.q_weight : p.k_weight;
      load_weights(weight, p.weight_bf16, l * 8, w);
      load_weights(weight, p.weight_bf16, kInterleaved ? l * 8 : partner_lane(l, p.rot) * 8, wp);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        a[e] *= w[e];
        b[e] *= wp[kInterleaved ? e ^ 1 : e];
      }
    }
  }
  for (int h = t.h0; h < t.h1; h += kUnroll) {
    uint4 x[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i)
      if (h + i < t.h1) x[i] = __ldg(reinterpret_cast<const uint4*>(src + (head_base + h + i) * kRow));
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      if (h + i >= t.h1) break;
      uint4 y = x[i];
      if (t.kind < 2) {
        float f[8], g[8];
        unpack8(x[i], f);
        unpack8(partner_of<kInterleaved>(x[i], src_lane), g);
        float r = 1.f;
        if (norm) {
          float sq = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) sq = fmaf(f[e], f[e], sq);
          r = rsqrtf(half_sum(sq) * (1.f / kRow) + p.eps);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = r * fmaf(g[e], b[e], f[e] * a[e]);
        y = pack8(f);
      }
      if (t.valid) *out_row(h + i) = y;
    }
  }
}

template <bool kInterleaved>
__global__ void __launch_bounds__(kThreadsRope) qkv_norm_rope_bwd_kernel(const __grid_constant__ RopeParams p) {
  __shared__ float sums[kWarps][2][kRow];
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x & 31, l = lane & 15, half = lane >> 4, warp = threadIdx.x >> 5;
  const int all_heads = p.heads + 2 * p.kv_heads;
  const bool norm = p.q_weight != nullptr;
  const int src_lane = half * 16 + partner_lane(l, p.rot);
  float dw[2][8];
#pragma unroll
  for (int e = 0; e < 8; ++e) dw[0][e] = dw[1][e] = 0.f;
  for (long long task = static_cast<long long>(blockIdx.x) * kWarps + warp; task < p.tasks;
       task += static_cast<long long>(gridDim.x) * kWarps) {
    const Task t = decode(p, task, half);
    const int head_base = t.kind == 0 ? 0 : (t.kind == 1 ? p.heads : p.heads + p.kv_heads);
    const int in_heads = t.kind == 0 ? p.heads : p.kv_heads;
    const __nv_bfloat16* const dy = t.kind == 0 ? p.q : (t.kind == 1 ? p.k : p.v);
    const __nv_bfloat16* const src = p.qkv + t.batch * p.stride_b + t.s * p.stride_s + l * 8;
    __nv_bfloat16* const dst = p.dqkv + static_cast<long long>(t.token) * all_heads * kRow + l * 8;
    auto in_row = [&](int h) {
      return reinterpret_cast<const uint4*>(
          dy + ((static_cast<long long>(t.batch) * in_heads + h) * p.seq + t.s) * kRow + l * 8);
    };
    float c[8], s[8], w[8];
    if (t.kind < 2) {
      load_turn<kInterleaved>(p, t, l, c, s);
      if (norm) load_weights(t.kind == 0 ? p.q_weight : p.k_weight, p.weight_bf16, l * 8, w);
    }
    for (int h = t.h0; h < t.h1; h += kUnroll) {
      uint4 d[kUnroll], x[kUnroll];
#pragma unroll
      for (int i = 0; i < kUnroll; ++i)
        if (h + i < t.h1) {
          d[i] = __ldg(in_row(h + i));
          if (t.kind < 2 && norm) x[i] = __ldg(reinterpret_cast<const uint4*>(src + (head_base + h + i) * kRow));
        }
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) {
        if (h + i >= t.h1) break;
        uint4 y = d[i];
        if (t.kind < 2) {
          float g[8], o[8];
          unpack8(d[i], g);
          unpack8(partner_of<kInterleaved>(d[i], src_lane), o);
#pragma unroll
          for (int e = 0; e < 8; ++e) g[e] = fmaf(-o[e], s[e], g[e] * c[e]);
          if (norm) {
            float f[8];
            unpack8(x[i], f);
            float sq = 0.f, dot = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              sq = fmaf(f[e], f[e], sq);
              dot = fmaf(g[e] * w[e], f[e], dot);
            }
            const float r = rsqrtf(half_sum(sq) * (1.f / kRow) + p.eps);
            const float m = half_sum(dot) * (1.f / kRow) * r;  // mean of g w x_hat
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float xh = f[e] * r;
              const float gx = t.valid ? g[e] * xh : 0.f;
              if (t.kind == 0) dw[0][e] += gx; else dw[1][e] += gx;
              g[e] = r * fmaf(-xh, m, g[e] * w[e]);
            }
          }
          y = pack8(g);
        }
        if (t.valid) *reinterpret_cast<uint4*>(dst + (head_base + h + i) * kRow) = y;
      }
    }
  }
  if (!norm) return;
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = dw[k][e] + __shfl_xor_sync(0xffffffffu, dw[k][e], 16);
      if (half == 0) sums[warp][k][l * 8 + e] = v;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * kRow; i += kThreadsRope) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) v += (&sums[k][0][0])[i];
    p.partial[static_cast<long long>(blockIdx.x) * (2 * kRow) + i] = v;
  }
}

// dw[col] = sum over CTAs of partial[cta][col]: 32 columns per block, 32 threads per column.
__global__ void __launch_bounds__(1024)
    weight_grad_kernel(const float* __restrict__ partial, int ctas, float* __restrict__ dq_weight,
                       float* __restrict__ dk_weight) {
  __shared__ float sums[32][33];
  grid_dependency_wait();
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), part = threadIdx.x >> 5;
  float v = 0.f;
  for (int c = part; c < ctas; c += 32) v += partial[static_cast<long long>(c) * (2 * kRow) + col];
  sums[part][threadIdx.x & 31] = v;
  __syncthreads();
  if (part == 0) {
    float total = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) total += sums[k][threadIdx.x];
    if (col < kRow)
      dq_weight[col] = total;
    else
      dk_weight[col - kRow] = total;
  }
}

}  // namespace rope
}  // namespace avo_b200
