// Attention of 1 to 16 query tokens over a KV cache held in 4 bits (format: cache4_sm100.cuh), sm_100a.
//
// Query t of T of sequence b sees rows j < kv_lens[b] - (T - 1 - t): the T queries are the sequence's last T tokens,
// whose rows are in the cache. Scale 1/8, FP32 softmax, query head h reads K/V head h / (Hq / Hkv); the
// G T rows of one K/V head are stacked, 8 or 16 of them to a tile.
//
// Products. Codes are never expanded to memory: a lane turns the words of its rows into halves in registers, where
// code x scale is exact, in the order in which mma.sync.m16n8k16 takes them. S^T = K Q^T and O^T = V^T P^T:
// 16 cached rows (features) are M, the 8 query rows N, so that a group of a few query heads wastes little (tcgen05
// takes its A operand from shared or tensor memory, at least 64 rows high: halves would have to be written there,
// four times the bytes that are read).
//   K: lane (g, t) = (lane / 4, lane % 4) holds features 16 t .. 16 t + 15, one scale group, of two rows:
//      8 bytes each. The features of a k-step are any 16 as long as Q's fragment has the same order.
//   S^T to P^T: rows in lanes to rows in registers, one movmatrix for 8 x 8.
//   V: pairs of adjacent tokens must share a register: the codes of two rows are interleaved (two shifts, two
//      selects for 16 values) before they are converted, not the halves after.
// Q is scaled by a power of two per row, its largest element to [2^14, 2^15), and held in half precision: 11
// significant bits over 2^28 against bf16's 8, so nothing is lost that is not 2^-36 of the row's largest element. P is
// rounded to half precision too: its rows are held below 2^15 by the running maximum, so that a weight is rounded by
// 2^-11 of itself down to 2^-29 of the largest one. Sums, maxima and the accumulators are FP32.
//
// Work. A warp takes tiles of 64 rows of one (sequence, K/V head, row tile), each by asynchronous copies into its own
// ring of shared memory, and keeps a softmax of its own; there is no barrier in the loop. The running maximum moves only
// when a tile exceeds it by 2^8 (a vote in place of a reduction). The warps of a CTA merge in shared memory, the
// CTAs of a cluster through distributed shared memory, and where one cluster is not enough for a
// long cache several write records that a second kernel merges.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "cache4_sm100.cuh"
#include "sm100_ptx.cuh"

namespace tt {
namespace cache4 {
namespace attn {

constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;
constexpr int TILE_BLOCKS = 4;
constexpr int TILE_ROWS = TILE_BLOCKS * BLOCK_ROWS;
constexpr int STAGES = 3;
constexpr int MAX_CLUSTER = 8;          // portable cluster size
constexpr int HALF_BYTES = TILE_BLOCKS * BLOCK_BYTES;   // K (or V) of a tile
constexpr int STAGE_BYTES = 2 * HALF_BYTES;
constexpr int CHUNKS = HALF_BYTES / 16;                 // 144 copies of 16 bytes
constexpr int LANE_CHUNKS = (CHUNKS + 31) / 32;
constexpr int REC = HD + 2;             // sums of a row: 64 features, reference exponent, total weight
constexpr float NEG_INF = -__builtin_huge_valf();
constexpr float LN2 = 0.69314718055994530942f;
constexpr float SLACK = 8.0f;           // a tile may exceed the running maximum by 2^8
constexpr float RAISE = 7.0f;           // weights are held 2^7 higher: at most 2^15 as halves

struct Params {
  const __nv_bfloat16* q;
  int64_t q_sb, q_sh, q_st;
  View cache[2];
  const int32_t* lens;      // optional [B]
  int B, Hkv, G, T;         // G query heads of a K/V head, T query tokens
  int row_tiles;            // tiles of the G T rows
  int blocks;               // capacity in blocks
  int cluster, parts;       // CTAs of a cluster, clusters of a unit
  __nv_bfloat16* o;         // [B, Hq, T, 64]
  float* lse;               // optional [B, Hq, T]
  float* records;           // parts > 1: [unit, part, 8 NT rows, REC]
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
               "{%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// 16 bytes from global to shared memory, zeros where `keep` is false (nothing is read then).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool keep) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(keep ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint2 lds_u2(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds_u8(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void sts_u8(uint32_t addr, uint32_t v) {
  asm volatile("st.shared.u8 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// Weight of a part with reference exponent e against the common one, 0 for an empty part.
__device__ __forceinline__ float part_weight(float e, float ref) {
  return e == NEG_INF ? 0.0f : ex2_approx(e - ref);
}

__device__ __forceinline__ void write_row(const Params& p, int64_t row, int d, float v0, float v1) {
  *reinterpret_cast<uint32_t*>(p.o + row * HD + d) = pack_bf16x2(v0, v1);
}

template <int NT>
struct alignas(16) Smem {
  union {
    uint8_t ring[STAGES][STAGE_BYTES];
    float own[8 * NT][REC];   // the warp's record, once its ring is empty
  } warp[WARPS];
  // Records of the rows that this CTA finishes (every cluster-th), from every CTA of the cluster: behind the ring, as
  // this CTA may still be in its loop when they arrive.
  float from[8 * NT + MAX_CLUSTER - 1][REC];
};

template <int NT>
__global__ void __launch_bounds__(THREADS, 3) attention_kernel(const __grid_constant__ Params p) {
  constexpr int ROWS = 8 * NT;
  extern __shared__ uint8_t smem_raw[];
  Smem<NT>& sm = *reinterpret_cast<Smem<NT>*>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int rank = static_cast<int>(blockIdx.x) % p.cluster;
  const int pc = static_cast<int>(blockIdx.x) / p.cluster;      // unit * parts + part
  const int part = pc % p.parts, unit = pc / p.parts;
  const int rt = unit % p.row_tiles, bh = unit / p.row_tiles;
  const int b = bh / p.Hkv, hk = bh % p.Hkv;
  const int rows = min(p.G * p.T - rt * ROWS, ROWS);
  const int workers = WARPS * p.cluster * p.parts;
  const int worker = (part * p.cluster + rank) * WARPS + warp;
  // Arrived at before the others' shared memory is written: a CTA that has not started has none.
  if (p.cluster > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  wait_for_previous_kernel();

  const int capacity = p.blocks * BLOCK_ROWS;
  const int len = p.lens != nullptr ? min(max(p.lens[b], 0), capacity) : capacity;
  const int tiles = (len + TILE_ROWS - 1) / TILE_ROWS;

  // Copies of this lane: chunk lane + 32 i of the K (V) tile.
  const uint8_t* base[2] = {p.cache[0].p + b * p.cache[0].sb + hk * p.cache[0].sh,
                            p.cache[1].p + b * p.cache[1].sb + hk * p.cache[1].sh};
  const uint32_t ring = smem_u32(sm.warp[warp].ring);
  auto load_tile = [&](int tile, int stage) {
    const uint32_t dst = ring + stage * STAGE_BYTES;
#pragma unroll
    for (int i = 0; i < LANE_CHUNKS; ++i) {
      const int c = lane + 32 * i;
      if (c >= CHUNKS) break;
      const int blk = c / (BLOCK_BYTES / 16), off = c % (BLOCK_BYTES / 16) * 16;
      // The chunk's first row: half a row of codes, or the scales of four rows.
      const int r = blk * BLOCK_ROWS + (off < CODE_BYTES ? off / 32 : (off - CODE_BYTES) / 4);
      const bool keep = tile * TILE_ROWS + r < len;
      const int64_t at = static_cast<int64_t>(tile) * TILE_BLOCKS + (keep ? blk : 0);
#pragma unroll
      for (int kv = 0; kv < 2; ++kv)
        copy16(dst + kv * HALF_BYTES + c * 16, base[kv] + at * p.cache[kv].sn + off, keep);
    }
  };
  int next = worker;
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) {
    if (next < tiles) load_tile(next, s);
    copy_commit();
    next += workers;
  }

  // Q as B fragments: query row n = g of each tile of 8, features 16 t4 .. + 15, and the factor that turns its products
  // into exponents of 2. The factors are needed for rows 2 t4 and 2 t4 + 1.
  uint32_t qf[NT][8];
  float factor[NT][2];
  int limit[NT][2];   // rows of the cache that query row 2 t4 + j sees
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = n * 8 + g;
    float x[16];
    float top = 0.0f;
    if (r < rows) {
      const int gr = rt * ROWS + r;
      const __nv_bfloat16* src = p.q + b * p.q_sb + (hk * p.G + gr / p.T) * p.q_sh + (gr % p.T) * p.q_st + 16 * t4;
      float lo[8], hi[8];
      norm_rope::unpack8(*reinterpret_cast<const uint4*>(src), lo);
      norm_rope::unpack8(*reinterpret_cast<const uint4*>(src + 8), hi);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = lo[i];
        x[i + 8] = hi[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(x[i]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // 2^(14 - exponent of top) in two factors: one may leave FP32's range. A row of zeros, or with an infinity (its
    // products are not finite whatever the factor), keeps 1.
    int e = static_cast<int>(__float_as_uint(top) >> 23) - 127;
    if (top == 0.0f || e == 128) e = 14;
    const float up0 = __uint_as_float(static_cast<uint32_t>(127 + (14 - e) / 2) << 23);
    const float up1 = __uint_as_float(static_cast<uint32_t>(127 + (14 - e) - (14 - e) / 2) << 23);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      qf[n][i] = pack_half2(x[2 * i] * up0 * up1, x[2 * i + 1] * up0 * up1);
    const float f = 0.125f * 1.44269504088896340736f / up0 / up1;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      factor[n][j] = __shfl_sync(0xffffffffu, f, (2 * t4 + j) * 4);
      const int gr = rt * ROWS + n * 8 + 2 * t4 + j;
      limit[n][j] = len - (p.T - 1 - gr % p.T);
    }
  }

  float acc[NT][4][4] = {};    // O^T: features 8 g + 2 i (+ 1 in 2, 3), query rows 2 t4, 2 t4 + 1
  float mx[NT][2], ref[NT][2], total[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      mx[n][j] = NEG_INF;   // running maximum, the same in all lanes of a column
      ref[n][j] = 0.0f;     // exponent that weights are relative to: mx - RAISE
      total[n][j] = 0.0f;   // this lane's rows only
    }

  int stage = 0;
  for (int tile = worker; tile < tiles; tile += workers) {
    copy_wait<STAGES - 2>();
    __syncwarp();
    // Into the stage of the step before, which every lane has left.
    if (next < tiles) load_tile(next, stage == 0 ? STAGES - 1 : stage - 1);
    copy_commit();
    next += workers;
    const uint32_t ks = ring + stage * STAGE_BYTES, vs = ks + HALF_BYTES;
    const int row0 = tile * TILE_ROWS;
    const bool tail = row0 + TILE_ROWS > len;
    if (tail) {
      // Scales of rows behind the last one came with the last group of four: anything may stand there.
      const int first = len - row0, last = (first + 3) & ~3;
      for (int i = lane; i < (last - first) * 2 * GROUPS; i += 32) {
        const int r = first + i / (2 * GROUPS), j = i % (2 * GROUPS);
        sts_u8((j < GROUPS ? ks : vs) + (r / BLOCK_ROWS) * BLOCK_BYTES + CODE_BYTES +
                   (r % BLOCK_ROWS) * GROUPS + j % GROUPS, 0);
      }
      __syncwarp();
    }
    // A value that is not finite, in a row that some queries see and others do not, would reach them all as 0 x NaN:
    // its group counts as zero in the product, and as NaN for those that see it. hidden: rows (from hidden0) of this
    // lane's group of features.
    uint32_t hidden = 0;
    const int hidden0 = max(row0, len - (p.T - 1));
    if (p.T > 1 && hidden0 < row0 + TILE_ROWS) {
      const int end = min(len, row0 + TILE_ROWS);
      for (int r = hidden0; r < end; ++r) {
        const int i = r - row0;
        if (lds_u8(vs + (i / BLOCK_ROWS) * BLOCK_BYTES + CODE_BYTES + (i % BLOCK_ROWS) * GROUPS + (g >> 1)) >
            MAX_SCALE_BYTE)
          hidden |= 1u << (r - hidden0);
      }
      __syncwarp();
      for (int r = hidden0; r < end; ++r) {
        const int i = r - row0;
        if ((hidden >> (r - hidden0)) & 1u)
          sts_u8(vs + (i / BLOCK_ROWS) * BLOCK_BYTES + CODE_BYTES + (i % BLOCK_ROWS) * GROUPS + (g >> 1), 0);
      }
      __syncwarp();
    }
    // ---- S^T: rows (g >> 1) + 4 (g & 1), and 8 more, of each block
    float s[TILE_BLOCKS][NT][4];
    const int kr = (g >> 1) + 4 * (g & 1);
#pragma unroll
    for (int j = 0; j < TILE_BLOCKS; ++j) {
      const uint32_t blk = ks + j * BLOCK_BYTES;
      uint32_t a[2][8];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int r = kr + 8 * half;
        const uint2 w = lds_u2(blk + r * (HD / 2) + t4 * 8);
        const uint32_t scale = scale_pair(lds_u8(blk + CODE_BYTES + r * GROUPS + t4));
        uint32_t x[4], y[4];
        decode8(w.x, x);
        decode8(w.y, y);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          a[half][i] = mul_half2(x[i], scale);
          a[half][4 + i] = mul_half2(y[i], scale);
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) s[j][n][i] = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma_f16(s[j][n], a[0][2 * k], a[1][2 * k], a[0][2 * k + 1], a[1][2 * k + 1], qf[n][2 * k],
                  qf[n][2 * k + 1]);
      }
    }
    // ---- exponents, masks, the running maximum
    bool over = false;
    float top[NT][2];
    const bool masked = row0 + TILE_ROWS > len - (p.T - 1);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      top[n][0] = top[n][1] = NEG_INF;
#pragma unroll
      for (int j = 0; j < TILE_BLOCKS; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float y = s[j][n][i] * factor[n][i & 1];
          if (masked && row0 + j * BLOCK_ROWS + kr + 8 * (i >> 1) >= limit[n][i & 1]) y = NEG_INF;
          s[j][n][i] = y;
          top[n][i & 1] = fmaxf(top[n][i & 1], y);
        }
      }
      over = over || top[n][0] > mx[n][0] + SLACK || top[n][1] > mx[n][1] + SLACK;
    }
    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float m = fmaxf(top[n][j], mx[n][j]);
#pragma unroll
          for (int d = 4; d < 32; d *= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
          const float old = ref[n][j];
          const bool empty = mx[n][j] == NEG_INF;
          mx[n][j] = m;
          ref[n][j] = m == NEG_INF ? 0.0f : m - RAISE;
          const float f = empty ? 1.0f : ex2_approx(old - ref[n][j]);   // empty: the sums are zero, or NaN
          total[n][j] *= f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            acc[n][i][j] *= f;
            acc[n][i][2 + j] *= f;
          }
        }
    }
    // ---- P^T as B fragments
    uint32_t pf[TILE_BLOCKS][NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < TILE_BLOCKS; ++j) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[i] = ex2_approx(s[j][n][i] - ref[n][i & 1]);
          total[n][i & 1] += e[i];
        }
        pf[j][n][0] = transpose8x8(pack_half2(e[0], e[1]));
        pf[j][n][1] = transpose8x8(pack_half2(e[2], e[3]));
      }
    // ---- O^T += V^T P^T
#pragma unroll
    for (int j = 0; j < TILE_BLOCKS; ++j) {
      const uint32_t blk = vs + j * BLOCK_BYTES;
      uint32_t a[2][8];   // tokens (t4, 4 + t4) and (8 + t4, 12 + t4); features 8 g + 2 i at i, + 1 at 4 + i
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int r = t4 + 8 * half;
        const uint32_t w0 = lds_u32(blk + r * (HD / 2) + g * 4);
        const uint32_t w1 = lds_u32(blk + (r + 4) * (HD / 2) + g * 4);
        const uint32_t s0 = lds_u8(blk + CODE_BYTES + r * GROUPS + (g >> 1));
        const uint32_t s1 = lds_u8(blk + CODE_BYTES + (r + 4) * GROUPS + (g >> 1));
        const uint32_t scale = (s0 << 7) | (s1 << 23);
        const uint32_t even = (w0 & 0x0f0f0f0fu) | ((w1 << 4) & 0xf0f0f0f0u);
        const uint32_t odd = ((w0 >> 4) & 0x0f0f0f0fu) | (w1 & 0xf0f0f0f0u);
        uint32_t x[4], y[4];
        decode8(even, x);
        decode8(odd, y);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          a[half][i] = mul_half2(x[i], scale);
          a[half][4 + i] = mul_half2(y[i], scale);
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          mma_f16(acc[n][i], a[0][i], a[0][4 + i], a[1][i], a[1][4 + i], pf[j][n][0], pf[j][n][1]);
    }
    if (hidden != 0) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          // Bits of the rows below this query's limit.
          const int seen = limit[n][j] - hidden0;
          if (seen > 0 && (hidden & ((2u << min(seen - 1, 30)) - 1u)) != 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              acc[n][i][j] = acc[n][i][2 + j] = __uint_as_float(0x7fffffffu);
          }
        }
    }
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
  copy_wait<0>();
  __syncwarp();

  // ---- this warp's record: [row][feature], reference exponent, total
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float sum = total[n][j];
#pragma unroll
      for (int d = 4; d < 32; d *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      float* rec = sm.warp[warp].own[n * 8 + 2 * t4 + j];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<float2*>(rec + 8 * g + 2 * i) = make_float2(acc[n][i][j], acc[n][i][2 + j]);
      if (g == 0) {
        // Weightless but not empty: NaN scores leave the maximum alone.
        rec[HD] = mx[n][j] == NEG_INF && sum == 0.0f ? NEG_INF : ref[n][j];
        rec[HD + 1] = sum;
      }
    }
  __syncthreads();
  // ---- the CTA's record, at the cluster's CTA that finishes the row: row r at rank r % cluster
  const bool alone = p.cluster == 1 && p.parts == 1;
  if (p.cluster > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  const int d = 2 * lane;
  for (int r = warp; r < rows; r += WARPS) {
    float m = NEG_INF, l = 0.0f, v0 = 0.0f, v1 = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) m = fmaxf(m, sm.warp[w].own[r][HD]);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = part_weight(sm.warp[w].own[r][HD], m);
      const float2 x = *reinterpret_cast<const float2*>(&sm.warp[w].own[r][d]);
      l += f * sm.warp[w].own[r][HD + 1];
      v0 += f * x.x;
      v1 += f * x.y;
    }
    if (alone) {
      const int64_t row = static_cast<int64_t>(bh) * p.G * p.T + rt * ROWS + r;
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      write_row(p, row, d, v0 * inv, v1 * inv);
      if (p.lse != nullptr && lane == 0) p.lse[row] = l == 0.0f ? NEG_INF : (m + __log2f(l)) * LN2;
      continue;
    }
    if (p.cluster == 1) {
      float* rec = p.records + (static_cast<int64_t>(pc) * ROWS + r) * REC;
      *reinterpret_cast<float2*>(rec + d) = make_float2(v0, v1);
      if (lane == 0) *reinterpret_cast<float2*>(rec + HD) = make_float2(m, l);
      continue;
    }
    const uint32_t dst = map_to_rank(smem_u32(sm.from[r / p.cluster * p.cluster + rank]),
                                     static_cast<uint32_t>(r % p.cluster));
    st_cluster_f32x2(dst + d * 4, v0, v1);
    if (lane == 0) st_cluster_f32x2(dst + HD * 4, m, l);
  }
  if (p.cluster == 1) return;
  __syncwarp();
  cluster_sync();
  for (int r = rank + p.cluster * warp; r < rows; r += p.cluster * WARPS) {
    const float(*from)[REC] = sm.from + r / p.cluster * p.cluster;
    float m = NEG_INF, l = 0.0f, v0 = 0.0f, v1 = 0.0f;
    for (int c = 0; c < p.cluster; ++c) m = fmaxf(m, from[c][HD]);
    for (int c = 0; c < p.cluster; ++c) {
      const float f = part_weight(from[c][HD], m);
      const float2 x = *reinterpret_cast<const float2*>(&from[c][d]);
      l += f * from[c][HD + 1];
      v0 += f * x.x;
      v1 += f * x.y;
    }
    if (p.parts > 1) {
      float* rec = p.records + (static_cast<int64_t>(pc) * ROWS + r) * REC;
      *reinterpret_cast<float2*>(rec + d) = make_float2(v0, v1);
      if (lane == 0) *reinterpret_cast<float2*>(rec + HD) = make_float2(m, l);
      continue;
    }
    const int64_t row = static_cast<int64_t>(bh) * p.G * p.T + rt * ROWS + r;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    write_row(p, row, d, v0 * inv, v1 * inv);
    if (p.lse != nullptr && lane == 0) p.lse[row] = l == 0.0f ? NEG_INF : (m + __log2f(l)) * LN2;
  }
}

// Merges the parts' records: one CTA a row, each warp every eighth part.
constexpr int COMBINE_WARPS = 8;

__global__ void __launch_bounds__(COMBINE_WARPS * 32)
    combine_kernel(const __grid_constant__ Params p, int tile_rows) {
  __shared__ float rec[COMBINE_WARPS][REC];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = 2 * lane;
  const int per_head = p.G * p.T;
  const int bh = static_cast<int>(blockIdx.x) / per_head, gr = static_cast<int>(blockIdx.x) % per_head;
  const int64_t unit = static_cast<int64_t>(bh) * p.row_tiles + gr / tile_rows;
  wait_for_previous_kernel();
  const float* src = p.records + (unit * p.parts * tile_rows + gr % tile_rows) * REC;
  float m = NEG_INF, l = 0.0f, v0 = 0.0f, v1 = 0.0f;
#pragma unroll 4
  for (int c = warp; c < p.parts; c += COMBINE_WARPS) {
    const float* x = src + static_cast<int64_t>(c) * tile_rows * REC;
    const float2 v = *reinterpret_cast<const float2*>(x + d);
    const float2 ml = *reinterpret_cast<const float2*>(x + HD);
    const float top = fmaxf(m, ml.x);
    const float f = part_weight(m, top), h = part_weight(ml.x, top);
    m = top;
    l = l * f + ml.y * h;
    v0 = v0 * f + v.x * h;
    v1 = v1 * f + v.y * h;
  }
  *reinterpret_cast<float2*>(&rec[warp][d]) = make_float2(v0, v1);
  if (lane == 0) *reinterpret_cast<float2*>(&rec[warp][HD]) = make_float2(m, l);
  __syncthreads();
  if (warp != 0) return;
  m = NEG_INF;
  l = v0 = v1 = 0.0f;
#pragma unroll
  for (int w = 0; w < COMBINE_WARPS; ++w) m = fmaxf(m, rec[w][HD]);
#pragma unroll
  for (int w = 0; w < COMBINE_WARPS; ++w) {
    const float f = part_weight(rec[w][HD], m);
    l += f * rec[w][HD + 1];
    v0 += f * rec[w][d];
    v1 += f * rec[w][d + 1];
  }
  const int64_t row = blockIdx.x;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  write_row(p, row, d, v0 * inv, v1 * inv);
  if (p.lse != nullptr && lane == 0) p.lse[row] = l == 0.0f ? NEG_INF : (m + __log2f(l)) * LN2;
}

}  // namespace attn
}  // namespace cache4
}  // namespace tt
