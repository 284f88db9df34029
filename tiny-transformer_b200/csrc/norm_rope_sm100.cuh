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
// inside a lane and the norm's sums take three shuffles. A warp's item is four tokens of up to sixteen heads of one
// kind (query, key or value): the tokens' rows of q and k are adjacent in the [B, H, T, 64] outputs, the weights are
// multiplied into the table rows once, and the next heads are loaded while these are computed. Arithmetic is on packed FP32
// pairs.
//
// Measured (B200, 4 x 4096 tokens of 12 + 12 + 12 heads): forward 16.4 us (100 MB, 6.1 TB/s), backward 37 us (201 MB, 5.4
// TB/s; it waits for loads: 20 warps an SM, and with registers for 24 it spilled and took 58), the weights' sums 4 us.
// With items of 4 or 6 heads the step took 62 and 59 us against 57.
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
constexpr int MAX_HEADS = 16;      // of an item
constexpr int BATCH = 4;           // heads in flight together
constexpr int SMALL_BATCH = 2;     // (backward: each with two rows to load; append)

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
  int total[3];               // items of each kind in all groups
  Divisor groups, each[3];    // divisions by the groups of a sequence, by items[]
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
  if (at < 0 || at > (int64_t(1) << 40)) return at < 0 && p.pos_st == 0 ? max(at, -(int64_t(1) << 40)) + t : -1;
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

  // Item `index` of kind k.
  __device__ __forceinline__ void set(const Common& p, int k, int index, int lane) {
    kind = k;
    const int bg = p.each[k].of(index);
    first = (index - bg * static_cast<int>(p.each[k].d)) * p.per_item;
    heads = min(p.per_item, (kind == 0 ? p.Hq : p.Hkv) - first);
    b = p.groups.of(bg);
    t = (bg - b * static_cast<int>(p.groups.d)) * ROWS + (lane >> 3);
    row = t < p.T;
  }
  __device__ __forceinline__ int head0(const Common& p) const {   // of the projection
    return first + (kind == 0 ? 0 : kind == 1 ? p.Hq : p.Hq + p.Hkv);
  }
};

// A lane's eight features as packed FP32 pairs: even features (0, 2), (4, 6), odd ones (1, 3), (5, 7), so that the
// two of a rotation stand in the same place of two registers.
struct Pairs {
  uint64_t e[2], o[2];

  __device__ __forceinline__ void unpack(const uint4& v) {
    e[0] = f2_pack(bf16_lo(v.x), bf16_lo(v.y));
    e[1] = f2_pack(bf16_lo(v.z), bf16_lo(v.w));
    o[0] = f2_pack(bf16_hi(v.x), bf16_hi(v.y));
    o[1] = f2_pack(bf16_hi(v.z), bf16_hi(v.w));
  }
  __device__ __forceinline__ void set(const float (&x)[E]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      e[i] = f2_pack(x[4 * i], x[4 * i + 2]);
      o[i] = f2_pack(x[4 * i + 1], x[4 * i + 3]);
    }
  }
  __device__ __forceinline__ uint4 pack() const {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float e0, e1, o0, o1;
      f2_unpack(e[i], e0, e1);
      f2_unpack(o[i], o0, o1);
      u[2 * i] = pack_bf16x2(e0, o0);
      u[2 * i + 1] = pack_bf16x2(e1, o1);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
  __device__ __forceinline__ void scale(float r) {
    const uint64_t r2 = f2_pack(r, r);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      e[i] = f2_mul(e[i], r2);
      o[i] = f2_mul(o[i], r2);
    }
  }
  __device__ __forceinline__ float dot(const Pairs& b) const {
    const uint64_t s = f2_add(f2_fma(e[1], b.e[1], f2_mul(e[0], b.e[0])), f2_fma(o[1], b.o[1], f2_mul(o[0], b.o[0])));
    float lo, hi;
    f2_unpack(s, lo, hi);
    return lo + hi;
  }
};

// Sum over the eight lanes of a row, in every one of them.
__device__ __forceinline__ float row_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  v += __shfl_xor_sync(0xffffffffu, v, 2);
  return v + __shfl_xor_sync(0xffffffffu, v, 4);
}

__device__ __forceinline__ float inverse_rms(const Pairs& x, float eps) {
  return rsqrtf(row_sum(x.dot(x)) * (1.0f / HD) + eps);
}

// The rotation with the weights in it: y_2i = x_2i ec + x_2i+1 os, y_2i+1 = x_2i es + x_2i+1 oc (x normed; os has
// the rotation's minus).
struct Coefficients {
  uint64_t ec[2], es[2], oc[2], os[2];

  template <bool NORM>
  __device__ __forceinline__ void set(const Common& p, int kind, const Turn& u, int lane8) {
    float w[E];
    if (NORM) load_weight(p, kind, lane8, w);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint64_t c = f2_pack(u.c[2 * i], u.c[2 * i + 1]), s = f2_pack(u.s[2 * i], u.s[2 * i + 1]);
      const uint64_t minus = f2_pack(-u.s[2 * i], -u.s[2 * i + 1]);
      const uint64_t we = NORM ? f2_pack(w[4 * i], w[4 * i + 2]) : f2_pack(1.0f, 1.0f);
      const uint64_t wo = NORM ? f2_pack(w[4 * i + 1], w[4 * i + 3]) : f2_pack(1.0f, 1.0f);
      ec[i] = f2_mul(we, c);
      es[i] = f2_mul(we, s);
      oc[i] = f2_mul(wo, c);
      os[i] = f2_mul(wo, minus);
    }
  }
  __device__ __forceinline__ Pairs turn(const Pairs& x) const {
    Pairs y;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      y.e[i] = f2_fma(x.e[i], ec[i], f2_mul(x.o[i], os[i]));
      y.o[i] = f2_fma(x.e[i], es[i], f2_mul(x.o[i], oc[i]));
    }
    return y;
  }
};

template <bool NORM>
__device__ __forceinline__ uint4 turn_row(const uint4& v, const Coefficients& k, float eps) {
  Pairs x;
  x.unpack(v);
  if (NORM) x.scale(inverse_rms(x, eps));
  return k.turn(x).pack();
}

// An item's rows, head by head: N of them are in registers while the next are on their way.
template <int N>
struct HeadRows {
  const __nv_bfloat16* src;   // of the batch in `now`
  int64_t step;               // elements from head to head
  int left;                   // heads from `now` on
  uint4 now[N], next[N];

  __device__ __forceinline__ static void load(uint4 (&v)[N], const __nv_bfloat16* from, int64_t step, int count) {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < count) v[j] = *reinterpret_cast<const uint4*>(from + j * step);
  }
  __device__ __forceinline__ void start(const __nv_bfloat16* from, int64_t by, int heads) {
    src = from;
    step = by;
    left = heads;
    load(now, src, step, left);
  }
  __device__ __forceinline__ void prefetch() { load(next, src + N * step, step, left - N); }
  __device__ __forceinline__ bool advance() {
    left -= N;
    src += N * step;
#pragma unroll
    for (int j = 0; j < N; ++j) now[j] = next[j];
    return left > 0;
  }
};

// Turns an item's heads. A row whose position is outside the table (or the cache) is zero.
template <bool NORM, int N>
__device__ __forceinline__ void turn_heads(HeadRows<N>& in, const Coefficients& k, float eps, __nv_bfloat16* dst,
                                           int64_t step, bool row, bool ok) {
  do {
    in.prefetch();
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (j >= in.left) break;
      const uint4 y = turn_row<NORM>(in.now[j], k, eps);
      if (row) *reinterpret_cast<uint4*>(dst) = ok ? y : make_uint4(0, 0, 0, 0);
      dst += step;
    }
  } while (in.advance());
}

// ------------------------------------------------------------------------------- forward

struct ForwardParams {
  Common c;
  __nv_bfloat16* out[2];  // q [B, Hq, T, 64], k [B, Hkv, T, 64]
};

template <bool NORM>
__global__ void __launch_bounds__(THREADS) forward_kernel(const __grid_constant__ ForwardParams fp) {
  const Common& p = fp.c;
  const int lane = threadIdx.x & 31, lane8 = lane & 7;
  int index = static_cast<int>(blockIdx.x) * WARPS + (threadIdx.x >> 5), kind = 0;
  wait_for_previous_kernel();
  if (index >= p.total[0]) {
    index -= p.total[0];
    kind = 1;
  }
  if (index >= p.total[kind]) return;  // whole warps
  Item it;
  it.set(p, kind, index, lane);
  const __nv_bfloat16* src = p.qkv + it.b * p.x_sb + static_cast<int64_t>(it.row ? it.t : 0) * p.x_st +
                             it.head0(p) * p.x_sh + lane8 * E;
  HeadRows<BATCH> in;
  in.start(src, p.x_sh, it.heads);
  const int64_t pos = it.row ? position_of(p, it.b, it.t) : 0;
  const bool ok = it.row && pos >= 0 && pos < p.table_len;
  if (it.row && !ok && lane8 == 0) atomicOr(&g_tt_status, TT_ERR_RANGE);
  Turn u;
  load_turn(p, ok ? pos : 0, lane8, u);
  Coefficients k;
  k.set<NORM>(p, it.kind, u, lane8);
  const int heads = it.kind == 0 ? p.Hq : p.Hkv;
  turn_heads<NORM>(in, k, static_cast<float>(p.eps),
                   fp.out[it.kind] + ((static_cast<int64_t>(it.b) * heads + it.first) * p.T + it.t) * HD + lane8 * E,
                   static_cast<int64_t>(p.T) * HD, it.row, ok);
}

// ------------------------------------------------------------------------------- backward

struct BackwardParams {
  Common c;
  int ctas[3];                         // CTAs for each kind of heads
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
  const int total = p.total[kind], stride = bp.ctas[kind] * WARPS;
  const __nv_bfloat16* const grad0 = bp.g[kind];
  const int64_t g_sb = bp.g_sb[kind], g_sh = bp.g_sh[kind], g_st = bp.g_st[kind];
  wait_for_previous_kernel();
  if (kind == 2) {
    for (int index = cta * WARPS + warp; index < total; index += stride) {
      Item it;
      it.set(p, 2, index, lane);
      if (!it.row) continue;
      const __nv_bfloat16* grad = grad0 + it.b * g_sb + it.first * g_sh + it.t * g_st + lane8 * E;
      __nv_bfloat16* dst =
          bp.dx + ((static_cast<int64_t>(it.b) * p.T + it.t) * heads + it.head0(p)) * HD + lane8 * E;
      if (grad0 == nullptr) {
        for (int h = 0; h < it.heads; ++h) *reinterpret_cast<uint4*>(dst + h * HD) = make_uint4(0, 0, 0, 0);
        continue;
      }
      HeadRows<BATCH> in;
      in.start(grad, g_sh, it.heads);
      do {
        in.prefetch();
#pragma unroll
        for (int j = 0; j < BATCH; ++j, dst += HD)
          if (j < in.left) *reinterpret_cast<uint4*>(dst) = in.now[j];
      } while (in.advance());
    }
    return;
  }
  Pairs w, dw;
  if (NORM) {
    float each[E];
    load_weight(p, kind, lane8, each);
    w.set(each);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) dw.e[i] = dw.o[i] = f2_pack(0.0f, 0.0f);
  for (int index = cta * WARPS + warp; index < total; index += stride) {
    Item it;
    it.set(p, kind, index, lane);
    const int64_t pos = it.row ? position_of(p, it.b, it.t) : 0;
    const bool ok = it.row && pos >= 0 && pos < p.table_len;
    if (it.row && !ok && lane8 == 0) atomicOr(&g_tt_status, TT_ERR_RANGE);
    const int64_t t = it.row ? it.t : 0;
    const __nv_bfloat16* src = p.qkv + it.b * p.x_sb + t * p.x_st + it.head0(p) * p.x_sh + lane8 * E;
    const __nv_bfloat16* grad = grad0 + it.b * g_sb + it.first * g_sh + t * g_st + lane8 * E;
    __nv_bfloat16* dst = bp.dx + ((static_cast<int64_t>(it.b) * p.T + t) * heads + it.head0(p)) * HD + lane8 * E;
    // A row outside the table was not turned but zeroed: its x and g count as zeros.
    constexpr int N = SMALL_BATCH;
    uint4 xv[N], gv[N];
    auto load = [&](uint4 (&x)[N], uint4 (&g)[N], int h0) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        x[j] = g[j] = make_uint4(0, 0, 0, 0);
        if (h0 + j < it.heads && ok) {
          x[j] = *reinterpret_cast<const uint4*>(src + (h0 + j) * p.x_sh);
          if (grad0 != nullptr) g[j] = *reinterpret_cast<const uint4*>(grad + (h0 + j) * g_sh);
        }
      }
    };
    load(xv, gv, 0);
    Turn u;
    load_turn(p, ok ? pos : 0, lane8, u);
    uint64_t c[2], s[2], minus[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      c[i] = f2_pack(u.c[2 * i], u.c[2 * i + 1]);
      s[i] = f2_pack(u.s[2 * i], u.s[2 * i + 1]);
      minus[i] = f2_pack(-u.s[2 * i], -u.s[2 * i + 1]);
    }
#pragma unroll 1
    for (int h0 = 0; h0 < it.heads; h0 += N) {
      uint4 xn[N], gn[N];
      load(xn, gn, h0 + N);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (h0 + j >= it.heads) break;
        Pairs x, gy, g;
        x.unpack(xv[j]);
        gy.unpack(gv[j]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          g.e[i] = f2_fma(gy.e[i], c[i], f2_mul(gy.o[i], s[i]));
          g.o[i] = f2_fma(gy.o[i], c[i], f2_mul(gy.e[i], minus[i]));
        }
        if (NORM) {
          const float rms = inverse_rms(x, static_cast<float>(p.eps));   // all lanes: it shuffles
          const float r = ok ? rms : 0.0f;
          x.scale(r);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            dw.e[i] = f2_fma(g.e[i], x.e[i], dw.e[i]);
            dw.o[i] = f2_fma(g.o[i], x.o[i], dw.o[i]);
            g.e[i] = f2_mul(g.e[i], w.e[i]);
            g.o[i] = f2_mul(g.o[i], w.o[i]);
          }
          const float dot = row_sum(g.dot(x)) * (-1.0f / HD);
          const uint64_t dot2 = f2_pack(dot, dot);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            g.e[i] = f2_fma(x.e[i], dot2, g.e[i]);
            g.o[i] = f2_fma(x.o[i], dot2, g.o[i]);
          }
          g.scale(r);
        }
        if (it.row) *reinterpret_cast<uint4*>(dst + (h0 + j) * HD) = g.pack();
      }
#pragma unroll
      for (int j = 0; j < N; ++j) {
        xv[j] = xn[j];
        gv[j] = gn[j];
      }
    }
  }
  if constexpr (NORM) {
    __shared__ float sums[WARPS * ROWS][HD];
    float* sum = &sums[warp * ROWS + (lane >> 3)][lane8 * E];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f2_unpack(dw.e[i], sum[4 * i], sum[4 * i + 2]);
      f2_unpack(dw.o[i], sum[4 * i + 1], sum[4 * i + 3]);
    }
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
