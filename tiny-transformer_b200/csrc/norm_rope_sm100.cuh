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
// inside a lane and the norm's sums take three shuffles. A warp's item is four tokens of up to four heads of one kind
// (query, key or value): the tokens' rows of q and k are adjacent in the [B, H, T, 64] outputs, all of an item's loads
// are in flight together, and the weights are multiplied into the table rows once for its heads.
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
constexpr int MAX_HEADS = 4;

// Division of n < 2^31 by a number known on the host (Granlund and Montgomery, 1994): a product and a shift.
struct Divisor {
  uint32_t d, multiply, shift;

  void set(uint32_t by) {
    d = by;
    shift = 0;
    while ((1ull << shift) < by) ++shift;
    multiply = static_cast<uint32_t>(((1ull << 32) * ((1ull << shift) - by)) / by + 1);
  }
  __device__ __forceinline__ int of(int n) const {
    return static_cast<int>((__umulhi(static_cast<uint32_t>(n), multiply) + static_cast<uint32_t>(n)) >> shift);
  }
};

// What a call of any of the kernels here and of the cache's append has in common.
struct Common {
  const __nv_bfloat16* qkv;
  int64_t x_sb, x_st, x_sh;   // element strides of qkv (batch, token, head)
  int B, T, Hq, Hkv;
  int per_item;               // heads of an item, at most MAX_HEADS
  int items[3];               // items of the query, key and value heads of a group of four tokens
  Divisor groups, per_group, each[3];   // divisions by groups, by all items of one, by those of a kind
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

__device__ __forceinline__ void unpack8(const uint4& v, float (&x)[E]) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = bf16_lo(u[i]);
    x[2 * i + 1] = bf16_hi(u[i]);
  }
}

__device__ __forceinline__ void load_weight(const Common& p, int kind, int lane8, float (&w)[E]) {
  if (p.w_f32) {
    const float* src = static_cast<const float*>(p.w[kind]) + lane8 * E;
    const float4 lo = *reinterpret_cast<const float4*>(src), hi = *reinterpret_cast<const float4*>(src + 4);
    w[0] = lo.x; w[1] = lo.y; w[2] = lo.z; w[3] = lo.w;
    w[4] = hi.x; w[5] = hi.y; w[6] = hi.z; w[7] = hi.w;
  } else {
    unpack8(*reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.w[kind]) + lane8 * E), w);
  }
}

// A warp's item.
struct Item {
  int b, t;          // sequence, this lane's token
  int kind;          // 0 query, 1 key, 2 value heads
  int first, heads;  // of its kind
  bool row;          // this lane's token is there

  __device__ __forceinline__ void set(const Common& p, int index, int lane) {
    const int bg = p.per_group.of(index);
    const int at = index - bg * static_cast<int>(p.per_group.d);
    const int k = at < p.items[0] ? 0 : at < p.items[0] + p.items[1] ? 1 : 2;
    set_kind(p, k, bg, at - (k == 0 ? 0 : k == 1 ? p.items[0] : p.items[0] + p.items[1]), lane);
  }
  // Item `at` of kind k in group bg.
  __device__ __forceinline__ void set_kind(const Common& p, int k, int bg, int at, int lane) {
    kind = k;
    first = at * p.per_item;
    heads = min(p.per_item, (kind == 0 ? p.Hq : p.Hkv) - first);
    b = p.groups.of(bg);
    t = (bg - b * static_cast<int>(p.groups.d)) * ROWS + (lane >> 3);
    row = t < p.T;
  }
  __device__ __forceinline__ int head0(const Common& p) const {   // of the projection
    return first + (kind == 0 ? 0 : kind == 1 ? p.Hq : p.Hq + p.Hkv);
  }
};

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

// The rotation with the weights in it: y_2i = x_2i ec - x_2i+1 os, y_2i+1 = x_2i es + x_2i+1 oc (x normed).
struct Coefficients {
  float ec[E / 2], es[E / 2], oc[E / 2], os[E / 2];

  template <bool NORM>
  __device__ __forceinline__ void set(const Common& p, int kind, const Turn& u, int lane8) {
    float w[E];
    if (NORM) load_weight(p, kind, lane8, w);
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      const float we = NORM ? w[2 * i] : 1.0f, wo = NORM ? w[2 * i + 1] : 1.0f;
      ec[i] = we * u.c[i];
      es[i] = we * u.s[i];
      oc[i] = wo * u.c[i];
      os[i] = wo * u.s[i];
    }
  }
};

template <bool NORM>
__device__ __forceinline__ uint4 turn_row(const uint4& v, const Coefficients& k, float eps) {
  float x[E], y[E];
  unpack8(v, x);
  const float r = NORM ? inverse_rms(x, eps) : 1.0f;
#pragma unroll
  for (int i = 0; i < E / 2; ++i) {
    const float a = x[2 * i] * r, b = x[2 * i + 1] * r;
    y[2 * i] = a * k.ec[i] - b * k.os[i];
    y[2 * i + 1] = a * k.es[i] + b * k.oc[i];
  }
  return pack8(y);
}

// ------------------------------------------------------------------------------- forward

struct ForwardParams {
  Common c;
  int total;              // items
  __nv_bfloat16* out[2];  // q [B, Hq, T, 64], k [B, Hkv, T, 64]
};

template <bool NORM>
__global__ void __launch_bounds__(THREADS) forward_kernel(const __grid_constant__ ForwardParams fp) {
  const Common& p = fp.c;
  const int lane = threadIdx.x & 31, lane8 = lane & 7;
  const int index = static_cast<int>(blockIdx.x) * WARPS + (threadIdx.x >> 5);
  wait_for_previous_kernel();
  if (index >= fp.total) return;  // whole warps
  Item it;
  it.set(p, index, lane);
  const __nv_bfloat16* src = p.qkv + it.b * p.x_sb + static_cast<int64_t>(it.row ? it.t : 0) * p.x_st +
                             it.head0(p) * p.x_sh + lane8 * E;
  uint4 v[MAX_HEADS];
#pragma unroll
  for (int h = 0; h < MAX_HEADS; ++h)
    if (h < it.heads) v[h] = *reinterpret_cast<const uint4*>(src + h * p.x_sh);
  const int64_t pos = it.row ? position_of(p, it.b, it.t) : 0;
  const bool ok = it.row && pos >= 0 && pos < p.table_len;
  if (it.row && !ok && lane8 == 0) atomicOr(&g_tt_status, TT_ERR_RANGE);
  Turn u;
  load_turn(p, ok ? pos : 0, lane8, u);
  Coefficients k;
  k.set<NORM>(p, it.kind, u, lane8);
  const int heads = it.kind == 0 ? p.Hq : p.Hkv;
  __nv_bfloat16* dst = fp.out[it.kind] +
                       ((static_cast<int64_t>(it.b) * heads + it.first) * p.T + it.t) * HD + lane8 * E;
#pragma unroll
  for (int h = 0; h < MAX_HEADS; ++h) {
    if (h >= it.heads) break;
    const uint4 y = turn_row<NORM>(v[h], k, static_cast<float>(p.eps));
    // A row whose position is outside the table is zero.
    if (it.row)
      *reinterpret_cast<uint4*>(dst + static_cast<int64_t>(h) * p.T * HD) = ok ? y : make_uint4(0, 0, 0, 0);
  }
}

// ------------------------------------------------------------------------------- backward

struct BackwardParams {
  Common c;
  int total[3], ctas[3];               // items of each kind of heads, and CTAs for them (0 where none)
  const __nv_bfloat16* g[3];           // dq, dk [B, H, T, 64] after the rotation, dv; NULL: zero
  int64_t g_sb[3], g_sh[3], g_st[3];
  __nv_bfloat16* dx;                   // [B, T, Hq + 2 Hkv, 64]
  float* partial;                      // [query and key CTAs, 64]: their sums of dw
  void* dw[2];                         // in the weights' type
};

// A CTA's items are of one kind. Query and key heads: dx, and dw summed over the CTA's rows in a fixed order, so
// that it does not depend on timing (registers, then shared memory). Value heads: dv copied.
template <bool NORM>
__global__ void __launch_bounds__(THREADS, 5) backward_kernel(const __grid_constant__ BackwardParams bp) {
  const Common& p = bp.c;
  const int lane = threadIdx.x & 31, lane8 = lane & 7, warp = threadIdx.x >> 5;
  const int heads = p.Hq + 2 * p.Hkv;
  int cta = static_cast<int>(blockIdx.x), kind = 0;
  while (cta >= bp.ctas[kind]) cta -= bp.ctas[kind++];
  const int total = bp.total[kind], stride = bp.ctas[kind] * WARPS;
  const __nv_bfloat16* const grad0 = bp.g[kind];
  const int64_t g_sb = bp.g_sb[kind], g_sh = bp.g_sh[kind], g_st = bp.g_st[kind];
  wait_for_previous_kernel();
  if (kind == 2) {
    for (int index = cta * WARPS + warp; index < total; index += stride) {
      Item it;
      const int bg = p.each[2].of(index);
      it.set_kind(p, 2, bg, index - bg * static_cast<int>(p.each[2].d), lane);
      if (!it.row) continue;
      const __nv_bfloat16* grad = grad0 + it.b * g_sb + it.first * g_sh + it.t * g_st + lane8 * E;
      __nv_bfloat16* dst =
          bp.dx + ((static_cast<int64_t>(it.b) * p.T + it.t) * heads + it.head0(p)) * HD + lane8 * E;
      uint4 v[MAX_HEADS];
#pragma unroll
      for (int h = 0; h < MAX_HEADS; ++h) {
        v[h] = make_uint4(0, 0, 0, 0);
        if (h < it.heads && grad0 != nullptr) v[h] = *reinterpret_cast<const uint4*>(grad + h * g_sh);
      }
#pragma unroll
      for (int h = 0; h < MAX_HEADS; ++h)
        if (h < it.heads) *reinterpret_cast<uint4*>(dst + h * HD) = v[h];
    }
    return;
  }
  float w[E], dw[E];
  if (NORM) load_weight(p, kind, lane8, w);
#pragma unroll
  for (int i = 0; i < E; ++i) dw[i] = 0.0f;
  for (int index = cta * WARPS + warp; index < total; index += stride) {
    Item it;
    const int bg = p.each[kind].of(index);
    it.set_kind(p, kind, bg, index - bg * static_cast<int>(p.each[kind].d), lane);
    const int64_t pos = it.row ? position_of(p, it.b, it.t) : 0;
    const bool ok = it.row && pos >= 0 && pos < p.table_len;
    if (it.row && !ok && lane8 == 0) atomicOr(&g_tt_status, TT_ERR_RANGE);
    const int64_t t = it.row ? it.t : 0;
    const __nv_bfloat16* src = p.qkv + it.b * p.x_sb + t * p.x_st + it.head0(p) * p.x_sh + lane8 * E;
    const __nv_bfloat16* grad = grad0 + it.b * g_sb + it.first * g_sh + t * g_st + lane8 * E;
    __nv_bfloat16* dst = bp.dx + ((static_cast<int64_t>(it.b) * p.T + t) * heads + it.head0(p)) * HD + lane8 * E;
    // A row outside the table was not turned but zeroed: its x and g count as zeros.
    uint4 xv[MAX_HEADS], gv[MAX_HEADS];
#pragma unroll
    for (int h = 0; h < MAX_HEADS; ++h) {
      xv[h] = gv[h] = make_uint4(0, 0, 0, 0);
      if (h < it.heads && ok) {
        xv[h] = *reinterpret_cast<const uint4*>(src + h * p.x_sh);
        if (grad0 != nullptr) gv[h] = *reinterpret_cast<const uint4*>(grad + h * g_sh);
      }
    }
    Turn u;
    load_turn(p, ok ? pos : 0, lane8, u);
#pragma unroll
    for (int h = 0; h < MAX_HEADS; ++h) {
      if (h >= it.heads) break;
      float x[E], gy[E], g[E], dx[E];
      unpack8(xv[h], x);
      unpack8(gv[h], gy);
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        g[2 * i] = gy[2 * i] * u.c[i] + gy[2 * i + 1] * u.s[i];
        g[2 * i + 1] = gy[2 * i + 1] * u.c[i] - gy[2 * i] * u.s[i];
      }
      if (NORM) {
        const float rms = inverse_rms(x, static_cast<float>(p.eps));   // all lanes: it shuffles
        const float r = ok ? rms : 0.0f;
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
          x[i] *= r;
          dw[i] = fmaf(g[i], x[i], dw[i]);
          g[i] *= w[i];
          dot = fmaf(g[i], x[i], dot);
        }
        dot = row_sum(dot) * (1.0f / HD);
#pragma unroll
        for (int i = 0; i < E; ++i) dx[i] = (g[i] - x[i] * dot) * r;
      } else {
#pragma unroll
        for (int i = 0; i < E; ++i) dx[i] = g[i];
      }
      if (it.row) *reinterpret_cast<uint4*>(dst + static_cast<int64_t>(h) * HD) = pack8(dx);
    }
  }
  if constexpr (NORM) {
    __shared__ float sums[WARPS * ROWS][HD];
#pragma unroll
    for (int i = 0; i < E; ++i) sums[warp * ROWS + (lane >> 3)][lane8 * E + i] = dw[i];
    __syncthreads();
    if (threadIdx.x < HD) {
      float s = 0.0f;
#pragma unroll
      for (int j = 0; j < WARPS * ROWS; ++j) s += sums[j][threadIdx.x];
      bp.partial[static_cast<int64_t>(blockIdx.x) * HD + threadIdx.x] = s;
    }
  }
}

// dw: the CTAs' sums, added in a fixed order. One block for eight of the 128 features; 64 threads a feature.
constexpr int REDUCE_FEATURES = 8;
constexpr int REDUCE_THREADS = 64;

__global__ void __launch_bounds__(REDUCE_THREADS * REDUCE_FEATURES)
    reduce_kernel(const __grid_constant__ BackwardParams bp) {
  __shared__ double part[REDUCE_THREADS][REDUCE_FEATURES + 1];
  const int f = threadIdx.x % REDUCE_FEATURES, j = threadIdx.x / REDUCE_FEATURES;
  const int at = blockIdx.x * REDUCE_FEATURES + f, kind = at / HD;
  const float* src = bp.partial + static_cast<int64_t>(kind == 0 ? 0 : bp.ctas[0]) * HD + at % HD;
  wait_for_previous_kernel();
  double s = 0.0;
#pragma unroll 8
  for (int i = j; i < bp.ctas[kind]; i += REDUCE_THREADS) s += src[static_cast<int64_t>(i) * HD];
  part[j][f] = s;
  __syncthreads();
  if (j >= 8) return;
#pragma unroll
  for (int i = 8; i < REDUCE_THREADS; i += 8) s += part[j + i][f];
  // The eight sums of a feature are in lanes f, f + 8, .. of two warps.
  part[j][f] = s;
  __syncwarp();
  asm volatile("bar.sync 1, 64;" ::: "memory");
  if (j != 0) return;
  for (int i = 1; i < 8; ++i) s += part[i][f];
  void* out = bp.dw[kind];
  if (bp.c.w_f32)
    static_cast<float*>(out)[at % HD] = static_cast<float>(s);
  else
    static_cast<__nv_bfloat16*>(out)[at % HD] = __float2bfloat16_rn(static_cast<float>(s));
}

}  // namespace norm_rope
}  // namespace tt
