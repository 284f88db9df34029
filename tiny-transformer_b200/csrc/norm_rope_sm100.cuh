// RMS norm of every query and key head with the rotary embedding in the same pass, forward and
// backward, for a fused QKV projection, sm_100a.
//
//   qkv [B, T, Hq + 2 Hkv, 64] bf16 (query heads, key heads, value heads)
//   x a query or key head of one token, w the weight of its kind, (c_i, s_i) the table row of its position:
//     r = 1 / sqrt(mean(x^2) + eps),   n = x r w,
//     y_2i = n_2i c_i - n_2i+1 s_i,    y_2i+1 = n_2i s_i + n_2i+1 c_i
//   backward, g = dL/dy turned back (the same rotation with -s):
//     dw += g x r (over all rows),     dx = r (g w - x r^2 mean(g w x))
//   Without weights there is no norm (n = x): the rotation alone. All of it in FP32, one rounding to bf16.
//
// Bound by memory: 128 bytes in and 128 out per head forward; backward reads x and dy and writes dx. Eight
// lanes hold a row, 16 bytes each, so a warp's loads and stores are 4 whole rows; the pairs of the rotation stay
// inside a lane and the norm's sums take three shuffles. A warp's four rows are four tokens of one head: their
// rows of q and k are adjacent in the [B, H, T, 64] outputs, and the table rows stay in registers while
// the warp goes through heads.
#pragma once

#include <cuda_bf16.h>
#include <cstdint>

#include "sm100_ptx.cuh"

namespace tt {
namespace norm_rope {

constexpr int HD = 64;
constexpr int PAIRS = HD / 2;
constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;
constexpr int ROWS = 4;   // tokens of a warp's step
constexpr int LANES = 8;  // lanes of a row
constexpr int E = HD / LANES;

// What a call of any of the kernels here and of the cache's append has in common.
struct Common {
  const __nv_bfloat16* qkv;
  int64_t x_sb, x_st, x_sh;   // element strides of qkv (batch, token, head)
  int B, T, Hq, Hkv;
  int heads_per_item;         // a warp's item: 4 tokens, this many heads
  int items_per_group;        // items of one group of 4 tokens
  const void* w[2];           // q and k weight [64], both NULL: no norm
  bool w_f32;                 // else bf16
  const float* cos;           // [table_len, 32]
  const float* sin;
  int64_t table_len;
  int64_t position;                // position of token 0 where position_dev is NULL
  const int64_t* position_dev;     // position of (b, t): position_dev[b * pos_sb + t * pos_st]
  int64_t pos_sb, pos_st;          //   and + t where pos_st is 0
  double eps;
};

__device__ __forceinline__ int64_t position_of(const Common& p, int b, int t) {
  if (p.position_dev == nullptr) return p.position + t;
  const int64_t at = p.position_dev[b * p.pos_sb + t * p.pos_st];
  return p.pos_st != 0 ? at : at + t;
}

struct Turn {  // a row's cos and sin, this lane's four pairs
  float c[E / 2], s[E / 2];
};

__device__ __forceinline__ void load_turn(const Common& p, int64_t pos, int lane8, Turn& u) {
  const float4 c = *reinterpret_cast<const float4*>(p.cos + pos * PAIRS + lane8 * (E / 2));
  const float4 s = *reinterpret_cast<const float4*>(p.sin + pos * PAIRS + lane8 * (E / 2));
  u.c[0] = c.x; u.c[1] = c.y; u.c[2] = c.z; u.c[3] = c.w;
  u.s[0] = s.x; u.s[1] = s.y; u.s[2] = s.z; u.s[3] = s.w;
}

__device__ __forceinline__ void load_weight(const Common& p, int kind, int lane8, float (&w)[E]) {
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int at = lane8 * E + i;
    w[i] = p.w[kind] == nullptr ? 1.0f
           : p.w_f32 ? static_cast<const float*>(p.w[kind])[at]
                     : __bfloat162float(static_cast<const __nv_bfloat16*>(p.w[kind])[at]);
  }
}

__device__ __forceinline__ void unpack8(const uint4& v, float (&x)[E]) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = bf16_lo(u[i]);
    x[2 * i + 1] = bf16_hi(u[i]);
  }
}

__device__ __forceinline__ uint4 pack8(const float (&y)[E]) {
  return make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]),
                    pack_bf16x2(y[6], y[7]));
}

// Sum over the eight lanes of a row, in every one of them.
__device__ __forceinline__ float row_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  v += __shfl_xor_sync(0xffffffffu, v, 2);
  return v + __shfl_xor_sync(0xffffffffu, v, 4);
}

__device__ __forceinline__ float inverse_rms(const float (&x)[E], float eps) {
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < E; ++i) ss = fmaf(x[i], x[i], ss);
  return rsqrtf(row_sum(ss) * (1.0f / HD) + eps);
}

// y = rotation of x r w (r = 1 and w = 1 without a norm).
__device__ __forceinline__ void turn_row(const float (&x)[E], const float (&w)[E], float r, const Turn& u,
                                         float (&y)[E]) {
#pragma unroll
  for (int i = 0; i < E / 2; ++i) {
    const float a = x[2 * i] * w[2 * i] * r, b = x[2 * i + 1] * w[2 * i + 1] * r;
    y[2 * i] = a * u.c[i] - b * u.s[i];
    y[2 * i + 1] = a * u.s[i] + b * u.c[i];
  }
}

// ------------------------------------------------------------------------------- forward

struct ForwardParams {
  Common c;
  __nv_bfloat16* q_out;   // [B, Hq, T, 64]
  __nv_bfloat16* k_out;   // [B, Hkv, T, 64]
};

template <bool NORM>
__global__ void __launch_bounds__(THREADS) forward_kernel(const __grid_constant__ ForwardParams fp) {
  const Common& p = fp.c;
  const int lane = threadIdx.x & 31, lane8 = lane & 7;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * WARPS + (threadIdx.x >> 5);
  const int groups = (p.T + ROWS - 1) / ROWS;
  wait_for_previous_kernel();
  if (item >= static_cast<int64_t>(p.B) * groups * p.items_per_group) return;  // whole warps
  const int64_t bg = item / p.items_per_group;
  const int first = static_cast<int>(item % p.items_per_group) * p.heads_per_item;
  const int last = min(first + p.heads_per_item, p.Hq + p.Hkv);
  const int b = static_cast<int>(bg / groups);
  const int t = static_cast<int>(bg % groups) * ROWS + (lane >> 3);
  const bool row = t < p.T;
  const int64_t pos = row ? position_of(p, b, t) : 0;
  const bool ok = row && pos >= 0 && pos < p.table_len;
  if (row && !ok && lane8 == 0) atomicOr(&g_tt_status, TT_ERR_RANGE);
  Turn u;
  load_turn(p, ok ? pos : 0, lane8, u);
  const __nv_bfloat16* src = p.qkv + b * p.x_sb + static_cast<int64_t>(row ? t : 0) * p.x_st + lane8 * E;
  float w[E];
  int kind = -1;
#pragma unroll 2
  for (int h = first; h < last; ++h) {
    const int now = h < p.Hq ? 0 : 1;
    if (NORM && now != kind) load_weight(p, now, lane8, w);
    kind = now;
    float x[E], y[E];
    unpack8(*reinterpret_cast<const uint4*>(src + h * p.x_sh), x);
    float r = 1.0f;
    if (NORM) {
      r = inverse_rms(x, static_cast<float>(p.eps));
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) w[i] = 1.0f;
    }
    turn_row(x, w, r, u, y);
    // A row whose position is outside the table is zero.
    const uint4 out = ok ? pack8(y) : make_uint4(0, 0, 0, 0);
    __nv_bfloat16* dst = now == 0 ? fp.q_out + ((static_cast<int64_t>(b) * p.Hq + h) * p.T + t) * HD
                                  : fp.k_out + ((static_cast<int64_t>(b) * p.Hkv + h - p.Hq) * p.T + t) * HD;
    if (row) *reinterpret_cast<uint4*>(dst + lane8 * E) = out;
  }
}

// ------------------------------------------------------------------------------- backward

struct BackwardParams {
  Common c;
  const __nv_bfloat16* g[3];           // dq, dk [B, H, T, 64] after the rotation, dv; NULL: zero
  int64_t g_sb[3], g_sh[3], g_st[3];
  __nv_bfloat16* dx;                   // [B, T, Hq + 2 Hkv, 64]
  float* partial;                      // [grid, 2, 64]: this CTA's sums of dw
  void* dw[2];                         // in the weights' type
  int blocks;
};

// dx of every head (a value head's gradient is copied), and per CTA the sum of dw over its rows, added in a
// fixed order so that it does not depend on timing: registers, then the CTA's rows through shared memory.
template <bool NORM>
__global__ void __launch_bounds__(THREADS) backward_kernel(const __grid_constant__ BackwardParams bp) {
  const Common& p = bp.c;
  const int lane = threadIdx.x & 31, lane8 = lane & 7, warp = threadIdx.x >> 5;
  const int groups = (p.T + ROWS - 1) / ROWS;
  const int heads = p.Hq + 2 * p.Hkv;
  const int64_t items = static_cast<int64_t>(p.B) * groups * p.items_per_group;
  wait_for_previous_kernel();
  float w[2][E], dw[2][E];
#pragma unroll
  for (int kind = 0; kind < 2; ++kind) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      w[kind][i] = 1.0f;
      dw[kind][i] = 0.0f;
    }
    if (NORM) load_weight(p, kind, lane8, w[kind]);
  }
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * WARPS + warp; item < items;
       item += static_cast<int64_t>(gridDim.x) * WARPS) {
    const int64_t bg = item / p.items_per_group;
    const int first = static_cast<int>(item % p.items_per_group) * p.heads_per_item;
    const int last = min(first + p.heads_per_item, heads);
    const int b = static_cast<int>(bg / groups);
    const int t = static_cast<int>(bg % groups) * ROWS + (lane >> 3);
    const bool row = t < p.T;
    const int64_t pos = row ? position_of(p, b, t) : 0;
    const bool ok = row && pos >= 0 && pos < p.table_len;
    if (row && !ok && lane8 == 0) atomicOr(&g_tt_status, TT_ERR_RANGE);
    Turn u;
    load_turn(p, ok ? pos : 0, lane8, u);
    const int tt = row ? t : 0;
    const __nv_bfloat16* src = p.qkv + b * p.x_sb + static_cast<int64_t>(tt) * p.x_st + lane8 * E;
    __nv_bfloat16* dst = bp.dx + ((static_cast<int64_t>(b) * p.T + tt) * heads) * HD + lane8 * E;
#pragma unroll 2
    for (int h = first; h < last; ++h) {
      const int part = h < p.Hq ? 0 : h < p.Hq + p.Hkv ? 1 : 2;
      const int hp = h - (part == 0 ? 0 : part == 1 ? p.Hq : p.Hq + p.Hkv);
      uint4 gv = make_uint4(0, 0, 0, 0);
      if (bp.g[part] != nullptr)
        gv = *reinterpret_cast<const uint4*>(bp.g[part] + b * bp.g_sb[part] + hp * bp.g_sh[part] +
                                             static_cast<int64_t>(tt) * bp.g_st[part] + lane8 * E);
      if (part == 2) {
        if (row) *reinterpret_cast<uint4*>(dst + static_cast<int64_t>(h) * HD) = gv;
        continue;
      }
      float x[E], gy[E], g[E];
      unpack8(*reinterpret_cast<const uint4*>(src + h * p.x_sh), x);
      unpack8(gv, gy);
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        // A row outside the table was not turned but zeroed: no gradient.
        const float a = ok ? gy[2 * i] : 0.0f, c = ok ? gy[2 * i + 1] : 0.0f;
        g[2 * i] = a * u.c[i] + c * u.s[i];
        g[2 * i + 1] = c * u.c[i] - a * u.s[i];
      }
      float dx[E];
      if (NORM) {
        const float r = inverse_rms(x, static_cast<float>(p.eps));
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const float n = x[i] * r;
          const float gw = g[i] * (part == 0 ? w[0][i] : w[1][i]);
          const float add = ok ? g[i] * n : 0.0f;
          if (part == 0) dw[0][i] += add; else dw[1][i] += add;
          x[i] = n;
          g[i] = gw;
          dot = fmaf(gw, n, dot);
        }
        dot = row_sum(dot) * (1.0f / HD);
#pragma unroll
        for (int i = 0; i < E; ++i) dx[i] = ok ? (g[i] - x[i] * dot) * r : 0.0f;
      } else {
#pragma unroll
        for (int i = 0; i < E; ++i) dx[i] = ok ? g[i] : 0.0f;
      }
      if (row) *reinterpret_cast<uint4*>(dst + static_cast<int64_t>(h) * HD) = pack8(dx);
    }
  }
  if constexpr (NORM) {
    __shared__ float sums[2][WARPS * ROWS][HD];
#pragma unroll
    for (int kind = 0; kind < 2; ++kind)
#pragma unroll
      for (int i = 0; i < E; ++i) sums[kind][warp * ROWS + (lane >> 3)][lane8 * E + i] = dw[kind][i];
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * HD; i += THREADS) {
      float s = 0.0f;
#pragma unroll
      for (int j = 0; j < WARPS * ROWS; ++j) s += sums[i / HD][j][i % HD];
      bp.partial[static_cast<int64_t>(blockIdx.x) * 2 * HD + i] = s;
    }
  }
}

// dw: the CTAs' sums, added in a fixed order. One block for eight of the 128 features; 32 threads a feature.
constexpr int REDUCE_FEATURES = 8;

__global__ void __launch_bounds__(32 * REDUCE_FEATURES)
    reduce_kernel(const __grid_constant__ BackwardParams bp) {
  __shared__ double part[32][REDUCE_FEATURES + 1];
  const int f = threadIdx.x % REDUCE_FEATURES, j = threadIdx.x / REDUCE_FEATURES;
  const int at = blockIdx.x * REDUCE_FEATURES + f;
  wait_for_previous_kernel();
  double s = 0.0;
#pragma unroll 4
  for (int i = j; i < bp.blocks; i += 32) s += bp.partial[static_cast<int64_t>(i) * 2 * HD + at];
  part[j][f] = s;
  __syncthreads();
  if (j != 0) return;
  for (int i = 1; i < 32; ++i) s += part[i][f];
  void* out = bp.dw[at / HD];
  if (bp.c.w_f32)
    static_cast<float*>(out)[at % HD] = static_cast<float>(s);
  else
    static_cast<__nv_bfloat16*>(out)[at % HD] = __float2bfloat16_rn(static_cast<float>(s));
}

}  // namespace norm_rope
}  // namespace tt
