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
// tree_attention_kernel<RT>: RT 16-row tiles (16 or 32 query rows) against tiles of 128 keys.
// One thread-block cluster takes one (batch, K/V head, row tile); its CTAs share the sequence's
// actual tiles evenly (tree tiles first, so rank 0 holds the mask), whatever the length. A
// producer warp keeps a ring of 128-key K and V tiles in flight with TMA (128-byte swizzle: 16-
// byte piece c of row r at piece c ^ (r % 8)); 4 consumer warps take 32 keys of a tile each, so
// that K and V fragments are read from shared memory once for all rows. Scores and P.V are
// mma.m16n8k16 on register fragments (Q stays in registers, P goes from the score fragments to
// the second product's A operand without leaving them); every warp keeps its own online softmax
// (m, l, O) and the CTA merges its warps at the end, the cluster its CTAs through distributed
// shared memory, each rank merging its share of the rows.
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
  const int32_t* parents;     // [N] (stride 0) or [B, N]
  int64_t parents_sb;
  const int32_t* lens;        // optional [B]
  int B, Hkv, G, N, C;
  int row_tiles;              // row tiles of one (batch, K/V head)
  int splits;                 // CTAs per cluster
  __nv_bfloat16* o;           // contiguous [B, G * Hkv, N, 64]
  float* lse;                 // optional [B, G * Hkv, N]
  float scale_log2;
};

template <int RT>
struct alignas(1024) Smem {
  static constexpr int ROWS = RT * 16;
  union {
    uint8_t ring[STAGES][2][TILE_BYTES];             // K and V tiles
    float rec[CONSUMER_WARPS][ROWS][REC];            // after the last tile: the warps' results
  };
  float crec[ROWS][REC];                             // the CTA's result, read by the cluster
  uint32_t mask[MAX_NODES][MASK_WORDS];              // bit m of row n: node n sees node m
  int32_t jump[MAX_NODES];
  uint64_t full[STAGES], empty[STAGES];
  int used[ROWS];                                    // rank 0: rows whose node is in use
  volatile int abort;
};
template <int RT>
constexpr size_t smem_bytes() { return sizeof(Smem<RT>); }

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
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ int ld_cluster_s32(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ int valid_len(const int32_t* lens, int C, int b) {
  if (lens == nullptr) return C;
  return min(max(__ldg(lens + b), 0), C);
}

// Ancestor masks of one tree from its parents, by doubling: mask[n] covers the chain from n up to,
// and without, jump[n]; a round ORs in the mask at jump[n] and jumps as far as that does, so a
// chain of any length takes log2(length) rounds. Links go to strictly lower indices (any other
// link ends the chain as unused, jump -2), so rounds go over blocks of `threads` nodes from the
// highest down, each reading before it writes, and never meet a node already updated this round.
// `sync` is a barrier of the `threads` threads that all call this; it returns whether any of them
// passed true.
template <typename Sync>
__device__ __forceinline__ void build_masks(const int32_t* parents, int N, int32_t* jump,
                                            uint32_t (*mask)[MASK_WORDS], int tid, int threads,
                                            Sync sync) {
  const int words = (N + 31) >> 5;
  bool more = false;
  for (int n = tid; n < N; n += threads) {
    const int up = __ldg(parents + n);
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

// One warp's state: Q fragments of RT row tiles, and the online softmax of its keys.
template <int RT>
struct WarpState {
  uint32_t qf[RT][4][4];   // A fragments of Q: 4 k-steps of 16 features
  float o[RT][8][4];       // O: 8 n-tiles of 8 features
  float m[RT][2], l[RT][2];
};

template <int RT>
__device__ __forceinline__ void reset(WarpState<RT>& st) {
#pragma unroll
  for (int t = 0; t < RT; ++t) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) st.o[t][j][e] = 0.f;
    st.m[t][0] = st.m[t][1] = -INFINITY;
    st.l[t][0] = st.l[t][1] = 0.f;
  }
}

template <int RT>
__device__ __forceinline__ void load_q(WarpState<RT>& st, const Params& p, int b, int h, int row0,
                                       int lane) {
#pragma unroll
  for (int t = 0; t < RT; ++t) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int r = row0 + t * 16 + half * 8 + (lane >> 2);
      const bool in = r < p.G * p.N;
      const int g = in ? r / p.N : 0, n = in ? r - g * p.N : 0;
      const uint32_t* src = reinterpret_cast<const uint32_t*>(
          p.q + b * p.q_sb + static_cast<int64_t>(h * p.G + g) * p.q_sh + n * p.q_sn) + (lane & 3);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        st.qf[t][k][half] = in ? __ldg(src + k * 8) : 0u;
        st.qf[t][k][half + 2] = in ? __ldg(src + k * 8 + 4) : 0u;
      }
    }
  }
}

// One warp's 32 keys of a tile: ks / vs are the shared addresses of its K and V rows (the first
// a multiple of 32 rows, so row % 8 is the swizzle phase), n_valid the rows that exist. TREE: the
// keys are tree nodes key0 .. key0 + 31 under the mask; otherwise every row sees every valid key.
template <int RT, bool TREE>
__device__ __forceinline__ void tile_step(WarpState<RT>& st, const Params& p, uint32_t ks,
                                          uint32_t vs, int n_valid, int lane,
                                          const uint32_t (*mask)[MASK_WORDS], int key0, int row0) {
  // V rows that no row may read: zeroed, so that 0 * (whatever they hold) stays 0.
  uint32_t bad = 0;  // TREE: keys in use whose V row holds an infinity or a NaN
  if (TREE || n_valid < 32) {
    bool clear = lane >= n_valid;
    if (TREE) clear = clear || !node_used(mask, key0 + lane);
    const uint32_t row = vs + lane * ROW_BYTES;
    if (clear) {
#pragma unroll
      for (int c = 0; c < 8; ++c) sts_u4(row + c * 16, 0, 0, 0, 0);
    } else if (TREE) {
      bool nf = false;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const uint4 u = lds_u4(row + c * 16);
        nf = nf || has_nonfinite(u.x) || has_nonfinite(u.y) || has_nonfinite(u.z) ||
             has_nonfinite(u.w);
      }
      bad = nf ? 1u : 0u;
    }
    if (TREE) bad = __ballot_sync(0xffffffffu, bad != 0);
    __syncwarp();
  }
  // S = Q K^T: 4 n-tiles of 8 keys. One ldmatrix.x4 holds 8 keys x 32 features (two k-steps).
  float s[RT][4][4];
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[t][j][e] = 0.f;
  const uint32_t kr = ks + (lane & 7) * ROW_BYTES;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      uint32_t bfr[4];
      ldmatrix_x4(kr + j * 8 * ROW_BYTES + (((kk * 4 + (lane >> 3)) ^ (lane & 7)) << 4), bfr);
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        mma_16816(s[t][j], st.qf[t][kk * 2], bfr[0], bfr[1]);
        mma_16816(s[t][j], st.qf[t][kk * 2 + 1], bfr[2], bfr[3]);
      }
    }
  }
  // Mask, running max and exponentials. Thread: rows lane / 4 and lane / 4 + 8 of each row tile,
  // keys 8 j + 2 (lane % 4) + {0, 1}.
  uint32_t pf[RT][4][2];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (TREE) {
        const int r = row0 + t * 16 + half * 8 + (lane >> 2);
        const uint32_t bits = r < p.G * p.N ? mask[r % p.N][key0 >> 5] : 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (!((bits >> (j * 8 + (lane & 3) * 2 + e)) & 1u)) s[t][j][half * 2 + e] = -INFINITY;
      } else if (n_valid < 32) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (j * 8 + (lane & 3) * 2 + e >= n_valid) s[t][j][half * 2 + e] = -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) mx = fmaxf(mx, fmaxf(s[t][j][half * 2], s[t][j][half * 2 + 1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float m_new = fmaxf(st.m[t][half], mx * p.scale_log2);
      const float base = m_new == -INFINITY ? 0.f : m_new;  // nothing visible yet: exp2(-inf) = 0
      const float f = ex2_approx(st.m[t][half] - base);
      st.m[t][half] = m_new;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p0 = ex2_approx(fmaf(s[t][j][half * 2], p.scale_log2, -base));
        const float p1 = ex2_approx(fmaf(s[t][j][half * 2 + 1], p.scale_log2, -base));
        sum += p0 + p1;
        pf[t][j][half] = pack_bf16x2(p0, p1);
      }
      st.l[t][half] = st.l[t][half] * f + sum;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        st.o[t][j][half * 2] *= f;
        st.o[t][j][half * 2 + 1] *= f;
      }
    }
  }
  if (TREE && bad != 0) {
    // Visible rows add p * v of these keys one by one; the V rows are then cleared.
    for (uint32_t left = bad; left != 0; left &= left - 1) {
      const int key = __ffs(left) - 1;
      const int src = (lane & ~3) | ((key & 7) >> 1);
      const uint32_t row = vs + key * ROW_BYTES;
#pragma unroll
      for (int t = 0; t < RT; ++t) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int r = row0 + t * 16 + half * 8 + (lane >> 2);
          const bool sees = r < p.G * p.N && ((mask[r % p.N][key0 >> 5] >> key) & 1u);
          uint32_t pair = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t x = __shfl_sync(0xffffffffu, pf[t][j][half], src);
            if (j == key >> 3) pair = x;
          }
          const float pr = (key & 1) ? bf16_hi(pair) : bf16_lo(pair);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint32_t v2 = lds_u32(row + ((j ^ (key & 7)) << 4) + (lane & 3) * 4);
            if (sees) {
              st.o[t][j][half * 2] = fmaf(pr, bf16_lo(v2), st.o[t][j][half * 2]);
              st.o[t][j][half * 2 + 1] = fmaf(pr, bf16_hi(v2), st.o[t][j][half * 2 + 1]);
            }
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
  // O += P V: two k-steps of 16 keys. One transposing ldmatrix.x4 holds 16 keys x 16 features.
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int key = k * 16 + (lane & 15);
    const uint32_t vr = vs + key * ROW_BYTES;
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) {
      uint32_t bfr[4];
      ldmatrix_x4_trans(vr + (((jj * 2 + (lane >> 4)) ^ (key & 7)) << 4), bfr);
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const uint32_t a[4] = {pf[t][2 * k][0], pf[t][2 * k][1], pf[t][2 * k + 1][0],
                               pf[t][2 * k + 1][1]};
        mma_16816(st.o[t][jj * 2], a, bfr[0], bfr[1]);
        mma_16816(st.o[t][jj * 2 + 1], a, bfr[2], bfr[3]);
      }
    }
  }
  // Zeroed rows were generic writes; the next TMA write of the stage is an asynchronous one.
  if (TREE || n_valid < 32) fence_proxy_async_smem();
}

// The warp's result into its record: O (not normalised), m and the full row sum l.
template <int RT>
__device__ __forceinline__ void store_record(WarpState<RT>& st, float (*rec)[REC], int lane) {
#pragma unroll
  for (int t = 0; t < RT; ++t) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float l = st.l[t][half];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      float* row = rec[t * 16 + half * 8 + (lane >> 2)];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        *reinterpret_cast<float2*>(row + j * 8 + (lane & 3) * 2) =
            make_float2(st.o[t][j][half * 2], st.o[t][j][half * 2 + 1]);
      if ((lane & 3) == 0) {
        row[HD] = st.m[t][half];
        row[HD + 1] = l;
      }
    }
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

template <int RT>
__global__ void __launch_bounds__(THREADS)
tree_attention_kernel(const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v,
                      const __grid_constant__ CUtensorMap tm_tk,
                      const __grid_constant__ CUtensorMap tm_tv, const Params p) {
  constexpr int ROWS = RT * 16;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem<RT>& s = *reinterpret_cast<Smem<RT>*>(smem_raw);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int unit = static_cast<int>(blockIdx.x) / p.splits;
  const int bh = unit / p.row_tiles;
  const int row0 = (unit - bh * p.row_tiles) * ROWS;
  const int b = bh / p.Hkv, h = bh - b * p.Hkv;
  const int L = valid_len(p.lens, p.C, b);
  const int tree_tiles = (p.N + KEYS - 1) / KEYS;
  const int tiles = tree_tiles + (L + KEYS - 1) / KEYS;
  const int first = static_cast<int>(static_cast<int64_t>(tiles) * rank / p.splits);
  const int last = static_cast<int>(static_cast<int64_t>(tiles) * (rank + 1) / p.splits);

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], CONSUMER_WARPS);
    }
    s.abort = 0;
    fence_barrier_init();
  }
  __syncthreads();

  if (warp == CONSUMER_WARPS) {
    // Producer: tile i into stage i % STAGES once the consumers have released it. Rows past the
    // tensor's end read as zero; rows past the length are loaded and never used.
    if (lane == 0) {
      int issued = 0;
      for (int i = first; i < last; ++i, ++issued) {
        const int st = issued % STAGES;
        if (issued >= STAGES && !wait_or_abort(&s.abort, &s.empty[st], ((issued / STAGES) + 1) & 1))
          break;
        mbar_arrive_expect_tx(&s.full[st], 2 * TILE_BYTES);
        if (i < tree_tiles) {
          tma_load_4d(s.ring[st][0], &tm_tk, &s.full[st], 0, i * KEYS, h, b);
          tma_load_4d(s.ring[st][1], &tm_tv, &s.full[st], 0, i * KEYS, h, b);
        } else {
          tma_load_4d(s.ring[st][0], &tm_k, &s.full[st], 0, (i - tree_tiles) * KEYS, h, b);
          tma_load_4d(s.ring[st][1], &tm_v, &s.full[st], 0, (i - tree_tiles) * KEYS, h, b);
        }
      }
      // Never leave while a TMA write into this CTA's shared memory is pending.
      if (s.abort)
        for (int c = max(0, issued - STAGES); c < issued; ++c)
          mbar_wait(&s.full[c % STAGES], (c / STAGES) & 1);
    }
    __syncwarp();
  } else {
    WarpState<RT> st;
    load_q(st, p, b, h, row0, lane);
    reset(st);
    if (first < tree_tiles || rank == 0) {
      build_masks(p.parents + b * p.parents_sb, p.N, s.jump, s.mask, threadIdx.x,
                  CONSUMER_WARPS * 32,
                  [](bool any) { return barrier_or<CONSUMER_WARPS * 32>(any); });
    }
    if (rank == 0 && threadIdx.x < ROWS) {
      const int r = row0 + static_cast<int>(threadIdx.x);
      s.used[threadIdx.x] = r < p.G * p.N && node_used(s.mask, r % p.N);
    }
    for (int i = first; i < last; ++i) {
      const int c = i - first, sg = c % STAGES;
      if (!warp_wait(&s.abort, &s.full[sg], (c / STAGES) & 1)) break;
      const bool is_tree = i < tree_tiles;
      const int key0 = (is_tree ? i : i - tree_tiles) * KEYS + warp * 32;
      const int n_valid = min(32, (is_tree ? p.N : L) - key0);
      if (n_valid > 0) {
        const uint32_t ks = smem_u32(s.ring[sg][0]) + warp * 32 * ROW_BYTES;
        const uint32_t vs = smem_u32(s.ring[sg][1]) + warp * 32 * ROW_BYTES;
        if (is_tree) tile_step<RT, true>(st, p, ks, vs, n_valid, lane, s.mask, key0, row0);
        else tile_step<RT, false>(st, p, ks, vs, n_valid, lane, s.mask, key0, row0);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.empty[sg]);
    }
    // Every tile of this CTA has landed and been read by all warps before the ring is reused.
    asm volatile("bar.sync 1, %0;" ::"n"(CONSUMER_WARPS * 32) : "memory");
    if (!s.abort) store_record(st, s.rec[warp], lane);
  }
  __syncthreads();

  // The CTA's warps: 8 threads a row, 8 features each.
  const int64_t out0 = static_cast<int64_t>(bh) * p.G * p.N + row0;
  const int rows = min(ROWS, p.G * p.N - row0);
  for (int i = threadIdx.x; i < rows * 8; i += THREADS) {
    const int r = i >> 3, c8 = i & 7;
    float M = -INFINITY, den = 0.f, n[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < CONSUMER_WARPS; ++w) M = fmaxf(M, s.rec[w][r][HD]);
#pragma unroll
    for (int w = 0; w < CONSUMER_WARPS; ++w) {
      const float wt = merge_weight(s.rec[w][r][HD], M);
      den = fmaf(wt, s.rec[w][r][HD + 1], den);
#pragma unroll
      for (int e = 0; e < 8; ++e) n[e] = fmaf(wt, s.rec[w][r][c8 * 8 + e], n[e]);
    }
    if (p.splits == 1) {
      write_out(p, out0 + r, c8, n, M, den, s.used[r] != 0);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) s.crec[r][c8 * 8 + e] = n[e];
      if (c8 == 0) {
        s.crec[r][HD] = M;
        s.crec[r][HD + 1] = den;
      }
    }
  }
  if (p.splits == 1) return;
  cluster_sync();
  // The cluster's CTAs: rank k merges rows k, k + splits, ...
  for (int i = threadIdx.x; i < rows * 8; i += THREADS) {
    const int r = (i >> 3) * p.splits + rank, c8 = i & 7;
    if (r >= rows) break;
    const uint32_t mine = smem_u32(s.crec[r]);
    float M = -INFINITY, den = 0.f, n[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int c = 0; c < p.splits; ++c)
      M = fmaxf(M, ld_cluster_f32(map_to_rank(mine, c) + HD * 4));
    for (int c = 0; c < p.splits; ++c) {
      const uint32_t src = map_to_rank(mine, c);
      const float wt = merge_weight(ld_cluster_f32(src + HD * 4), M);
      den = fmaf(wt, ld_cluster_f32(src + (HD + 1) * 4), den);
      const float4 x = ld_cluster_f4(src + c8 * 32), y = ld_cluster_f4(src + c8 * 32 + 16);
      n[0] = fmaf(wt, x.x, n[0]); n[1] = fmaf(wt, x.y, n[1]);
      n[2] = fmaf(wt, x.z, n[2]); n[3] = fmaf(wt, x.w, n[3]);
      n[4] = fmaf(wt, y.x, n[4]); n[5] = fmaf(wt, y.y, n[5]);
      n[6] = fmaf(wt, y.z, n[6]); n[7] = fmaf(wt, y.w, n[7]);
    }
    write_out(p, out0 + r, c8, n, M, den,
              ld_cluster_s32(map_to_rank(smem_u32(&s.used[r]), 0)) != 0);
  }
  cluster_sync();  // no CTA leaves while another reads its records
}

}  // namespace tree
}  // namespace tt
