// Attention of a tree of drafted tokens over a KV cache for sm_100a (speculative decoding).
//
// Node n of sequence b attends to the cached prefix and to its own branch:
//   A(n) = {n, parent(n), parent(parent(n)), ...} up to a root (parent -1),
//   O[n] = softmax over {cache rows j < len_b} and {tree rows j in A(n)} of (q_n . k_j / 8) v_j,
// FP32 softmax, BF16 O, natural-log FP32 LSE. A node is in use when its chain reaches -1 over
// strictly lower indices; any other node (padding of a smaller tree) gets O = 0, LSE = -inf and
// is visible to nobody. What is not visible never contributes, whatever it holds: scores are
// selected to -inf, V rows that no row of the tile may read are zeroed before the products, and
// tree V rows holding infinities or NaN are added under the mask instead of multiplied by zero.
//
// The heads that share a K/V head are stacked: row r = g * N + n of the G * N query rows of one
// (batch, K/V head), so the cache is read once for all of them. The operator does 2 * G * N
// products per cached element and is bound by reading the cache for the trees it is made for.
//
// tree_attention_kernel: trees of at most 32 nodes, 16 stacked query rows at a time. One thread-block
// cluster takes one (batch, K/V head, 16 rows); its CTAs share the sequence's actual 128-key cache
// tiles evenly, whatever the length. A producer warp keeps a two-stage ring of K and V tiles in flight with TMA
// (128-byte swizzle: 16-byte piece c of row r at piece c ^ (r % 8)); 4 consumer warps take 32 keys
// of a tile each, so that K and V fragments are read from shared memory once. Scores and P.V are
// mma.m16n8k16 on register fragments (Q stays in registers, P goes from the score fragments to the
// second product's A operand without leaving them). P is rounded to BF16 for that product, the only
// rounding below 32 bits before the output's: it is what the tensor cores take beside a BF16 V, and what
// the framework's other attention kernels do. It adds up to 2^-8 of each weight; measured against 64
// bits, the outputs' relative error is 0.0020-0.0023, of which 0.00165 is the output's own rounding. Sums
// take P before it is rounded. The tree's keys are a step or two of rank 0's
// first warp, 16 keys each, loaded with plain loads under the first tiles' flight. Every warp keeps its own online
// softmax (m, l, O); the CTA merges its warps, every CTA pushes each row to the rank that owns it
// (st.shared::cluster), and after one cluster barrier each rank merges and writes its rows. 75 KiB
// of shared memory and 128 registers leave room for three CTAs per SM (192 KiB of loads in flight).
// Larger trees, and more rows over long caches (which would be read once per 16 rows), take
// tree_persistent_sm100.cuh.
//
// Measured (B200, 12 heads): 142 us, 6.42 TB/s, for 64 sequences of 1024-8192 cached rows and 16 nodes
// (99 % of the copy rate; 923 MB of DRAM reads for 911 MB of operands); 18.1 us, 4.2 TB/s, for 32
// sequences of 512-1024 rows and one node (384 short CTAs on 148 SMs: some SMs have three, some two, a
// sixth of the time; the rest above the memory's 11.7 us is their start and end); 6.8 us
// for 8 sequences of 256-512 rows and 16 nodes, 4.6 us for one of 320 rows and 8 nodes (latency: one
// tile's flight, four warps' step, the merges and one cluster barrier).
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cstdint>

#include "sm100_ptx.cuh"

namespace tt {
namespace tree {

constexpr int HD = 64;
constexpr int MAX_NODES = 256;
constexpr int MASK_WORDS = MAX_NODES / 32;
constexpr int CONSUMER_WARPS = 4;
constexpr int THREADS = (CONSUMER_WARPS + 1) * 32;
constexpr int KEYS = CONSUMER_WARPS * 32;             // keys per tile
constexpr uint32_t ROW_BYTES = HD * 2;
constexpr uint32_t TILE_BYTES = KEYS * ROW_BYTES;     // 16 KiB of K (and of V)
constexpr int STAGES = 2;
constexpr int MAX_SPLITS = 8;                         // portable cluster size
constexpr int REC = HD + 4;                           // O[64], m (log2 units), l, 2 pad
constexpr float LN2 = 0.69314718055994530942f;

struct Params {
  const __nv_bfloat16* q;
  int64_t q_sb, q_sh, q_sn;   // element strides of q [B, G * Hkv, N, 64]
  const __nv_bfloat16* tk;    // the tree's K and V [B, Hkv, N, 64]
  const __nv_bfloat16* tv;
  int64_t tk_sb, tk_sh, tk_sn, tv_sb, tv_sh, tv_sn;
  const int32_t* parents;     // [N] (stride 0) or [B, N]
  int64_t parents_sb;
  const int32_t* lens;        // optional [B]
  int B, Hkv, G, N, C;
  int row_tiles;              // row tiles of one (batch, K/V head)
  int splits;                 // cluster kernel: CTAs per cluster
  __nv_bfloat16* o;           // contiguous [B, G * Hkv, N, 64]
  float* lse;                 // optional [B, G * Hkv, N]
  float scale_log2;
};

constexpr int ROWS = 16;                              // query rows of a unit
constexpr int CLUSTER_NODES = 32;                     // nodes of a tree, cluster kernel
constexpr int PUSH_ROWS = 24;                         // splits * ceil(ROWS / splits) at most

struct alignas(1024) Smem {
  union {
    uint8_t ring[STAGES][2][TILE_BYTES];              // K and V tiles
    float rec[CONSUMER_WARPS][ROWS][REC];             // after the last tile: the warps' results
  };
  float push[PUSH_ROWS][REC];                         // this rank's rows from every CTA
  uint8_t tree[2][16 * ROW_BYTES];                    // rank 0: K and V rows of 16 nodes
  uint64_t full[STAGES], empty[STAGES];
  volatile int abort;
};
constexpr size_t kSmemBytes = sizeof(Smem);
// With the 1 KiB that the system takes of each, three CTAs fill the SM's 228 KiB exactly (two CTAs per
// SM: 14.2 instead of 7.4 us for 8 sequences of 256-512 rows).
static_assert(3 * (kSmemBytes + 1024) <= 228 * 1024, "three CTAs per SM");

// Bounded wait that gives up as soon as another warp of the CTA has given up.
__device__ __forceinline__ bool wait_or_abort(volatile int* abort, uint64_t* bar, uint32_t parity) {
  const uint32_t addr = smem_u32(bar);
  if (mbar_try_wait(addr, parity)) return true;
  const long long t0 = clock64();
  while (true) {
    if (mbar_try_wait(addr, parity)) return true;
    if (*abort) return false;
    if (clock64() - t0 > kWaitBudgetCycles) {
      atomicOr(&g_tt_status, TT_ERR_TIMEOUT);
      *abort = 1;
      return false;
    }
  }
}
__device__ __forceinline__ bool warp_wait(volatile int* abort, uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, wait_or_abort(abort, bar, parity));
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// D (16x8, FP32) += A (16x16) B (16x8), bf16 operands.
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ int valid_len(const int32_t* lens, int C, int b) {
  if (lens == nullptr) return C;
  return min(max(lens[b], 0), C);
}

// Ancestor masks of one tree from its parents, by doubling: mask[n] covers the chain from n up to,
// and without, jump[n]; a round ORs in the mask at jump[n] and jumps as far as that does, so a
// chain of any length takes log2(length) rounds. Links go to strictly lower indices (any other
// link ends the chain as unused, jump -2), so rounds go over blocks of `threads` nodes from the
// highest down, each reading before it writes, and never meet a node that its round has updated.
// `sync` is a barrier of the `threads` threads that all call this; it returns whether any of them
// passed true.
template <typename Sync>
__device__ __forceinline__ void build_masks(const int32_t* parents, int N, int32_t* jump,
                                            uint32_t (*mask)[MASK_WORDS], int tid, int threads,
                                            Sync sync) {
  const int words = (N + 31) >> 5;
  bool more = false;
  for (int n = tid; n < N; n += threads) {
    const int up = parents[n];
    jump[n] = up < n && up >= -1 ? up : -2;
    more = more || (up < n && up >= 0);
    for (int w = 0; w < MASK_WORDS; ++w) mask[n][w] = w == n >> 5 ? 1u << (n & 31) : 0u;
  }
  while (sync(more)) {
    more = false;
    for (int base = (N - 1) / threads * threads; base >= 0; base -= threads) {
      const int n = base + tid;
      const int j = n < N ? jump[n] : -1;
      int far = j;
      uint32_t add[MASK_WORDS];
      if (j >= 0) {
        far = jump[j];
#pragma unroll
        for (int w = 0; w < MASK_WORDS; ++w) add[w] = w < words ? mask[j][w] : 0u;
      }
      sync(false);
      if (j >= 0) {
        jump[n] = far;
#pragma unroll
        for (int w = 0; w < MASK_WORDS; ++w)
          if (w < words) mask[n][w] |= add[w];
        more = more || far >= 0;
      }
    }
  }
  for (int n = tid; n < N; n += threads)
    if (jump[n] != -1)
      for (int w = 0; w < MASK_WORDS; ++w) mask[n][w] = 0;
  sync(false);
}

__device__ __forceinline__ bool node_used(const uint32_t (*mask)[MASK_WORDS], int n) {
  return (mask[n][n >> 5] >> (n & 31)) & 1u;
}

__device__ __forceinline__ bool has_nonfinite(uint32_t u) {
  return (u & 0x7F80u) == 0x7F80u || (u & 0x7F800000u) == 0x7F800000u;
}

// Named barrier 1 of `THREADS_` threads; whether any of them passed true.
template <int THREADS_>
__device__ __forceinline__ bool barrier_or(bool any) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred.aligned q, 1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r) : "r"(any ? 1u : 0u), "n"(THREADS_) : "memory");
  return r != 0;
}

// One warp's state: Q fragments, and the online softmax of its keys.
struct WarpState {
  uint32_t qf[4][4];   // A fragments of Q: 4 k-steps of 16 features
  float o[8][4];       // O: 8 n-tiles of 8 features
  float m[2], l[2];    // rows lane / 4 and lane / 4 + 8
};

__device__ __forceinline__ void load_q(WarpState& st, const Params& p, int b, int h, int row0,
                                       int lane) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = row0 + half * 8 + (lane >> 2);
    const bool in = r < p.G * p.N;
    const int g = in ? r / p.N : 0, n = in ? r - g * p.N : 0;
    const uint32_t* src = reinterpret_cast<const uint32_t*>(
        p.q + b * p.q_sb + static_cast<int64_t>(h * p.G + g) * p.q_sh + n * p.q_sn) + (lane & 3);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      st.qf[k][half] = in ? src[k * 8] : 0u;
      st.qf[k][half + 2] = in ? src[k * 8 + 4] : 0u;
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) st.o[j][e] = 0.f;
  st.m[0] = st.m[1] = -INFINITY;
  st.l[0] = st.l[1] = 0.f;
}

// One warp's KEYS_ keys (32 of a cache tile, or the tree's 16): ks / vs are the shared addresses of
// its K and V rows (the first a multiple of 8 rows, so row % 8 is the swizzle phase). see[half]: the
// keys that row lane / 4 + 8 half sees. bad: keys whose V row holds infinities or NaN (tree only);
// their products are added under the mask, and the rows must not reach the matrix product.
template <int KEYS_>
__device__ __forceinline__ void tile_step(WarpState& st, float scale_log2, uint32_t ks, uint32_t vs,
                                          bool masked, const uint32_t (&see)[2], uint32_t bad,
                                          int lane) {
  constexpr int NT = KEYS_ / 8;
  // S = Q K^T: n-tiles of 8 keys. One ldmatrix.x4 holds 8 keys x 32 features (two k-steps).
  float s[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[j][e] = 0.f;
  const uint32_t kr = ks + (lane & 7) * ROW_BYTES;
#pragma unroll
  for (int j = 0; j < NT; ++j) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      uint32_t bfr[4];
      ldmatrix_x4(kr + j * 8 * ROW_BYTES + (((kk * 4 + (lane >> 3)) ^ (lane & 7)) << 4), bfr);
      mma_16816(s[j], st.qf[kk * 2], bfr[0], bfr[1]);
      mma_16816(s[j], st.qf[kk * 2 + 1], bfr[2], bfr[3]);
    }
  }
  // Mask, running max and exponentials. Thread: rows lane / 4 and lane / 4 + 8, keys
  // 8 j + 2 (lane % 4) + {0, 1}.
  uint32_t pf[NT][2];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    if (masked) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (!((see[half] >> (j * 8 + (lane & 3) * 2 + e)) & 1u)) s[j][half * 2 + e] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < NT; ++j) mx = fmaxf(mx, fmaxf(s[j][half * 2], s[j][half * 2 + 1]));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const float m_new = fmaxf(st.m[half], mx * scale_log2);
    const float base = m_new == -INFINITY ? 0.f : m_new;  // nothing visible yet: exp2(-inf) = 0
    const float f = ex2_approx(st.m[half] - base);
    st.m[half] = m_new;
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const float p0 = ex2_approx(fmaf(s[j][half * 2], scale_log2, -base));
      const float p1 = ex2_approx(fmaf(s[j][half * 2 + 1], scale_log2, -base));
      sum += p0 + p1;
      pf[j][half] = pack_bf16x2(p0, p1);
    }
    st.l[half] = st.l[half] * f + sum;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      st.o[j][half * 2] *= f;
      st.o[j][half * 2 + 1] *= f;
    }
  }
  if (bad != 0) {
    // Visible rows add p * v of these keys one by one; the V rows are then cleared.
    for (uint32_t left = bad; left != 0; left &= left - 1) {
      const int key = __ffs(left) - 1;
      const int src = (lane & ~3) | ((key & 7) >> 1);
      const uint32_t row = vs + key * ROW_BYTES;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t pair = 0;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint32_t x = __shfl_sync(0xffffffffu, pf[j][half], src);
          if (j == key >> 3) pair = x;
        }
        const float pr = (key & 1) ? bf16_hi(pair) : bf16_lo(pair);
        if ((see[half] >> key) & 1u) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint32_t v2 = lds_u32(row + ((j ^ (key & 7)) << 4) + (lane & 3) * 4);
            st.o[j][half * 2] = fmaf(pr, bf16_lo(v2), st.o[j][half * 2]);
            st.o[j][half * 2 + 1] = fmaf(pr, bf16_hi(v2), st.o[j][half * 2 + 1]);
          }
        }
      }
    }
    __syncwarp();
    if ((bad >> lane) & 1u) {
#pragma unroll
      for (int c = 0; c < 8; ++c) sts_u4(vs + lane * ROW_BYTES + c * 16, 0, 0, 0, 0);
    }
    __syncwarp();
  }
  // O += P V: k-steps of 16 keys. One transposing ldmatrix.x4 holds 16 keys x 16 features.
#pragma unroll
  for (int k = 0; k < NT / 2; ++k) {
    const int key = k * 16 + (lane & 15);
    const uint32_t vr = vs + key * ROW_BYTES;
    const uint32_t a[4] = {pf[2 * k][0], pf[2 * k][1], pf[2 * k + 1][0], pf[2 * k + 1][1]};
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) {
      uint32_t bfr[4];
      ldmatrix_x4_trans(vr + (((jj * 2 + (lane >> 4)) ^ (key & 7)) << 4), bfr);
      mma_16816(st.o[jj * 2], a, bfr[0], bfr[1]);
      mma_16816(st.o[jj * 2 + 1], a, bfr[2], bfr[3]);
    }
  }
}

// The warp's result into its record: O (not normalised), m and the full row sum l.
__device__ __forceinline__ void store_record(const WarpState& st, float (*rec)[REC], int lane) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    float l = st.l[half];
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    float* row = rec[half * 8 + (lane >> 2)];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      *reinterpret_cast<float2*>(row + j * 8 + (lane & 3) * 2) =
          make_float2(st.o[j][half * 2], st.o[j][half * 2 + 1]);
    if ((lane & 3) == 0) *reinterpret_cast<float2*>(row + HD) = make_float2(st.m[half], l);
  }
}

// Weights of merged partial softmaxes are exp2(m_i - M); a part that saw nothing has m = -inf.
__device__ __forceinline__ float merge_weight(float m, float M) {
  return m == -INFINITY ? 0.f : ex2_approx(m - M);
}

// Output of one 8-feature group of one row: den == 0 only where nothing was visible.
__device__ __forceinline__ void write_out(const Params& p, int64_t out_row, int c8,
                                          const float (&n)[8], float M, float den, bool used) {
  const float inv = (used && den != 0.f) ? 1.f / den : 0.f;
  uint4 u = make_uint4(0, 0, 0, 0);
  if (used && den != 0.f)
    u = make_uint4(pack_bf16x2(n[0] * inv, n[1] * inv), pack_bf16x2(n[2] * inv, n[3] * inv),
                   pack_bf16x2(n[4] * inv, n[5] * inv), pack_bf16x2(n[6] * inv, n[7] * inv));
  reinterpret_cast<uint4*>(p.o + out_row * HD)[c8] = u;
  if (c8 == 0 && p.lse != nullptr)
    p.lse[out_row] = (used && den != 0.f) ? (M + log2f(den)) * LN2 : -INFINITY;
}

// The step over 16 of the tree's own keys, from node `key0` on, by one warp: their K and V rows into
// shared memory (rows that are not in use as zeros), then the products under the ancestor masks.
// chain: lane n holds node n's mask.
__device__ __forceinline__ void tree_step(WarpState& st, const Params& p, Smem& s, int b, int h,
                                          int row0, int key0, uint32_t chain, uint32_t used,
                                          int lane) {
  const int c = lane & 7;
  uint4 k[4], v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = key0 + i * 4 + (lane >> 3);
    k[i] = v[i] = make_uint4(0, 0, 0, 0);
    if (n < p.N && ((used >> n) & 1u)) {
      k[i] = reinterpret_cast<const uint4*>(p.tk + b * p.tk_sb + h * p.tk_sh + n * p.tk_sn)[c];
      v[i] = reinterpret_cast<const uint4*>(p.tv + b * p.tv_sb + h * p.tv_sh + n * p.tv_sn)[c];
    }
  }
  const uint32_t ks = smem_u32(s.tree[0]), vs = smem_u32(s.tree[1]);
  uint32_t bad = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = i * 4 + (lane >> 3);
    const uint32_t at = n * ROW_BYTES + ((c ^ (n & 7)) << 4);
    sts_u4(ks + at, k[i].x, k[i].y, k[i].z, k[i].w);
    sts_u4(vs + at, v[i].x, v[i].y, v[i].z, v[i].w);
    const unsigned nf = __ballot_sync(0xffffffffu, has_nonfinite(v[i].x) || has_nonfinite(v[i].y) ||
                                                       has_nonfinite(v[i].z) || has_nonfinite(v[i].w));
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (nf & (0xFFu << (8 * r))) bad |= 1u << (i * 4 + r);
  }
  __syncwarp();
  uint32_t see[2];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = row0 + half * 8 + (lane >> 2);
    const uint32_t bits = __shfl_sync(0xffffffffu, chain, r % p.N);
    see[half] = r < p.G * p.N ? bits >> key0 : 0u;
  }
  tile_step<16>(st, p.scale_log2, ks, vs, true, see, bad, lane);
  __syncwarp();  // every lane has read the rows before the next step's
}

// MULTI: several row tiles per K/V head, or more than 16 nodes. (An instantiation of its own: carrying
// both costs the one-tile kernel 5 % on long caches. At 128 registers it spills 32 bytes, the other 4.)
template <bool MULTI>
__global__ void __launch_bounds__(THREADS, 3)
tree_attention_kernel(const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const Params p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem& s = *reinterpret_cast<Smem*>(smem_raw);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int unit = static_cast<int>(blockIdx.x) / p.splits;
  const int bh = MULTI ? unit / p.row_tiles : unit;
  const int row0 = MULTI ? (unit - bh * p.row_tiles) * ROWS : 0;
  const int b = bh / p.Hkv, h = bh - b * p.Hkv;
  const int rows = MULTI ? min(ROWS, p.G * p.N - row0) : p.G * p.N;
  wait_for_previous_kernel();
  const int L = valid_len(p.lens, p.C, b);
  const int tiles = (L + KEYS - 1) / KEYS;
  const int first = static_cast<int>(static_cast<int64_t>(tiles) * rank / p.splits);
  const int last = static_cast<int>(static_cast<int64_t>(tiles) * (rank + 1) / p.splits);
  // No CTA writes another's shared memory before that CTA has started (waited for at the end).
  if (p.splits > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

  // Producer: tile i into stage i % STAGES once the consumers have released it; the first tiles go
  // out before the CTA meets. Rows past the capacity read as zero; rows past the length are loaded
  // and never used.
  auto issue = [&](int i) {
    const int st = (i - first) % STAGES;
    mbar_arrive_expect_tx(&s.full[st], 2 * TILE_BYTES);
    tma_load_4d(s.ring[st][0], &tm_k, &s.full[st], 0, i * KEYS, h, b);
    tma_load_4d(s.ring[st][1], &tm_v, &s.full[st], 0, i * KEYS, h, b);
  };
  WarpState st;
  uint32_t chain = 0, used = 0;
  if (warp == CONSUMER_WARPS) {
    if (lane == 0) {
      for (int i = 0; i < STAGES; ++i) {
        mbar_init(&s.full[i], 1);
        mbar_init(&s.empty[i], CONSUMER_WARPS);
      }
      s.abort = 0;
      fence_barrier_init();
      for (int i = first; i < min(last, first + STAGES); ++i) issue(i);
    }
    __syncwarp();
  } else {
    load_q(st, p, b, h, row0, lane);
    // Ancestor mask of node `lane`, by climbing: links go to lower indices, so 32 steps at most.
    const int32_t* parents = p.parents + b * p.parents_sb;
    const int up = lane < p.N ? parents[lane] : -2;
    const int link = up < lane && up >= -1 ? up : -2;
    int at = lane;
    while (__any_sync(0xffffffffu, at >= 0)) {
      if (at >= 0) chain |= 1u << at;
      const int next = __shfl_sync(0xffffffffu, link, at & 31);
      if (at >= 0) at = next;
    }
    if (at != -1) chain = 0;
    used = __ballot_sync(0xffffffffu, chain != 0);
  }
  __syncthreads();

  if (warp == CONSUMER_WARPS) {
    if (lane == 0) {
      int issued = min(last, first + STAGES);
      for (; issued < last; ++issued) {
        const int k = issued - first;
        if (!wait_or_abort(&s.abort, &s.empty[k % STAGES], ((k / STAGES) + 1) & 1)) break;
        issue(issued);
      }
      // Never leave while a TMA write into this CTA's shared memory is pending.
      if (s.abort)
        for (int k = max(0, issued - first - STAGES); k < issued - first; ++k)
          mbar_wait(&s.full[k % STAGES], (k / STAGES) & 1);
    }
    __syncwarp();
  } else {
    if (rank == 0 && warp == 0)
      for (int key0 = 0; key0 < (MULTI ? p.N : 1); key0 += 16)
        tree_step(st, p, s, b, h, row0, key0, chain, used, lane);
    for (int i = first; i < last; ++i) {
      const int c = i - first, sg = c % STAGES;
      if (!warp_wait(&s.abort, &s.full[sg], (c / STAGES) & 1)) break;
      const int n_valid = min(32, L - i * KEYS - warp * 32);
      if (n_valid > 0) {
        const uint32_t ks = smem_u32(s.ring[sg][0]) + warp * 32 * ROW_BYTES;
        const uint32_t vs = smem_u32(s.ring[sg][1]) + warp * 32 * ROW_BYTES;
        const uint32_t all = n_valid < 32 ? (1u << n_valid) - 1u : 0xffffffffu;
        const uint32_t see[2] = {all, all};
        if (n_valid < 32) {
          // V rows past the length: zeroed, so that 0 * (whatever they hold) stays 0.
          if (lane >= n_valid) {
#pragma unroll
            for (int k = 0; k < 8; ++k) sts_u4(vs + lane * ROW_BYTES + k * 16, 0, 0, 0, 0);
          }
          __syncwarp();
        }
        tile_step<32>(st, p.scale_log2, ks, vs, n_valid < 32, see, 0u, lane);
        // (No TMA write follows the generic ones: a partial tile is the sequence's last.)
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.empty[sg]);
    }
    // Every tile of this CTA has landed and been read by all warps before the ring is reused.
    asm volatile("bar.sync 1, %0;" ::"n"(CONSUMER_WARPS * 32) : "memory");
    if (!s.abort) store_record(st, s.rec[warp], lane);
    asm volatile("bar.sync 1, %0;" ::"n"(CONSUMER_WARPS * 32) : "memory");
  }

  // The CTA's warps: 8 threads a row, 8 features each; then row r goes to rank r % splits.
  const int r = static_cast<int>(threadIdx.x) >> 3, c8 = threadIdx.x & 7;
  const bool task = warp < CONSUMER_WARPS && r < rows;
  float M = -INFINITY, den = 0.f, n[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  auto add = [&](const float* rec, float weight) {
    const float4 x = reinterpret_cast<const float4*>(rec)[c8 * 2];
    const float4 y = reinterpret_cast<const float4*>(rec)[c8 * 2 + 1];
    n[0] = fmaf(weight, x.x, n[0]); n[1] = fmaf(weight, x.y, n[1]);
    n[2] = fmaf(weight, x.z, n[2]); n[3] = fmaf(weight, x.w, n[3]);
    n[4] = fmaf(weight, y.x, n[4]); n[5] = fmaf(weight, y.y, n[5]);
    n[6] = fmaf(weight, y.z, n[6]); n[7] = fmaf(weight, y.w, n[7]);
  };
  if (task) {
    float2 ml[CONSUMER_WARPS];
#pragma unroll
    for (int w = 0; w < CONSUMER_WARPS; ++w) {
      ml[w] = *reinterpret_cast<const float2*>(s.rec[w][r] + HD);
      M = fmaxf(M, ml[w].x);
    }
#pragma unroll
    for (int w = 0; w < CONSUMER_WARPS; ++w) {
      const float weight = merge_weight(ml[w].x, M);
      den = fmaf(weight, ml[w].y, den);
      add(s.rec[w][r], weight);
    }
  }
  const int64_t out0 = static_cast<int64_t>(bh) * p.G * p.N + row0;
  if (p.splits == 1) {
    if (task) write_out(p, out0 + r, c8, n, M, den, (used >> ((row0 + r) % p.N)) & 1u);
    return;
  }
  __syncwarp();  // .aligned barriers take whole warps
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  const int each = (ROWS + p.splits - 1) / p.splits;  // rows a rank owns
  if (task) {
    const uint32_t dst =
        map_to_rank(smem_u32(s.push[rank * each + r / p.splits]), static_cast<uint32_t>(r % p.splits));
    st_cluster_v4(dst + c8 * 32, __float_as_uint(n[0]), __float_as_uint(n[1]), __float_as_uint(n[2]),
                  __float_as_uint(n[3]));
    st_cluster_v4(dst + c8 * 32 + 16, __float_as_uint(n[4]), __float_as_uint(n[5]),
                  __float_as_uint(n[6]), __float_as_uint(n[7]));
    if (c8 == 0) st_cluster_f32x2(dst + HD * 4, M, den);
  }
  __syncwarp();
  cluster_sync();
  // The cluster's CTAs, for this rank's rows. Nothing is written to another CTA any more.
  const int own = r * p.splits + rank;
  if (warp >= CONSUMER_WARPS || r >= each || own >= rows) return;
  M = -INFINITY;
  den = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) n[e] = 0.f;
  for (int k = 0; k < p.splits; ++k) M = fmaxf(M, s.push[k * each + r][HD]);
  for (int k = 0; k < p.splits; ++k) {
    const float* rec = s.push[k * each + r];
    const float2 ml = *reinterpret_cast<const float2*>(rec + HD);
    const float weight = merge_weight(ml.x, M);
    den = fmaf(weight, ml.y, den);
    add(rec, weight);
  }
  write_out(p, out0 + own, c8, n, M, den, (used >> ((row0 + own) % p.N)) & 1u);
}

}  // namespace tree
}  // namespace tt
