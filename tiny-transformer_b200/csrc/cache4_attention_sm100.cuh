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
// rounded to half precision too: its largest weight is held between 2^7 and 2^15 by the running maximum, so that a weight is
// rounded by 2^-11 of itself down to 2^-21 of the largest one, and is off by 2^-32 of the largest at most below that. V is
// scaled exactly and has no part in this. Sums, maxima and the accumulators are FP32.
//
// Work. A warp takes tiles of 64 rows of one (sequence, K/V head, row tile), each by asynchronous copies into its own
// ring of shared memory (two stages: a third took shared memory from other CTAs, 49.1 against 46.5 us on the case below),
// and keeps a softmax of its own; there is no barrier in the loop. The running maximum moves only when a tile exceeds it
// by 2^8 (a vote in place of a reduction). Two kernels share the work: a cluster for each unit (its CTAs merge through
// distributed shared memory; for few units and long caches several clusters or CTAs write records that a second
// kernel merges), and for many tiles the flat kernel below.
//
// Measured (B200, us in a CUDA graph): 64 sequences of 1024-8192 rows, 12 heads 49.7 (5.1 TB/s; 512 sequences 334,
// 6.1 TB/s); 32 x 8 K/V heads, 32 query heads, 1024-4096 rows 18.2 (2.6 TB/s); 2 K/V heads of 131072 rows 10.6;
// 12 heads of 512 rows 3.8. Long runs are bound by instruction issue (per 16 rows about 140 instructions with one query row,
// 160 with more: 32 conversions, 16 or 32 multiplications by scales, 8 products; 2.6 a cycle and SM), hundreds of long
// sequences with one query row by DRAM, short runs by start, merge and launch.
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
constexpr int STAGES = 2;
constexpr int MIN_CTAS = 4;             // CTAs of an SM
constexpr int MAX_CLUSTER = 8;          // portable cluster size
constexpr int HALF_BYTES = TILE_BLOCKS * BLOCK_BYTES;   // K (or V) of a tile
constexpr int STAGE_BYTES = 2 * HALF_BYTES;
constexpr int CHUNKS = HALF_BYTES / 16;                 // copies of 16 bytes
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
  int cluster, parts;       // CTAs of a cluster, clusters of a unit (cluster kernel)
  __nv_bfloat16* o;         // [B, Hq, T, 64]
  float* lse;               // optional [B, Hq, T]
  int2* parts_of;           // flat kernel: of each unit that has tiles, its first worker and their number
  float* records;           // [slot, 8 NT rows, REC]; cluster kernel: slot = unit * parts + part
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
               "{%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The first product of a sum.
__device__ __forceinline__ void mma_f16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                              uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
               "{%8, %9}, {%10, %10, %10, %10};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// 16 bytes from global to shared memory.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// The same, or zeros where `keep` is false (nothing is read then).
__device__ __forceinline__ void copy16_or_zero(uint32_t dst, const void* src, bool keep) {
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
__device__ __forceinline__ uint32_t lds_u16(uint32_t addr) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void sts_u8(uint32_t addr, uint32_t v) {
  asm volatile("st.shared.u8 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

__device__ __forceinline__ int visible_rows(const Params& p, int b) {
  const int capacity = p.blocks * BLOCK_ROWS;
  return p.lens != nullptr ? min(max(p.lens[b], 0), capacity) : capacity;
}

// One (sequence, K/V head, tile of query rows).
struct Unit {
  int b, hk, rt;
  int len, tiles;
  const uint8_t* base[2];

  __device__ __forceinline__ void set(const Params& p, int b_, int hk_, int rt_, int len_) {
    b = b_;
    hk = hk_;
    rt = rt_;
    len = len_;
    tiles = (len + TILE_ROWS - 1) / TILE_ROWS;
    base[0] = p.cache[0].p + b * p.cache[0].sb + hk * p.cache[0].sh;
    base[1] = p.cache[1].p + b * p.cache[1].sb + hk * p.cache[1].sh;
  }
};

// A warp's copies of one tile (K, then V) to a stage of its ring. `dense`: blocks follow each other in memory.
__device__ __forceinline__ void load_tile(const Params& p, const Unit& u, int tile, uint32_t dst, int lane,
                                          bool dense) {
  if (dense && (tile + 1) * TILE_ROWS <= u.len) {
    const int64_t at = static_cast<int64_t>(tile) * HALF_BYTES + lane * 16;
    const uint8_t* k = u.base[0] + at;
    const uint8_t* v = u.base[1] + at;
    dst += lane * 16;
#pragma unroll
    for (int i = 0; i < LANE_CHUNKS; ++i) {
      if (i * 32 + 32 > CHUNKS && lane + 32 * i >= CHUNKS) break;
      copy16(dst + i * 512, k + i * 512);
      copy16(dst + HALF_BYTES + i * 512, v + i * 512);
    }
    return;
  }
#pragma unroll 1
  for (int c = lane; c < CHUNKS; c += 32) {
    const int blk = c / (BLOCK_BYTES / 16), off = c % (BLOCK_BYTES / 16) * 16;
    // The chunk's first row: half a row of codes, or the scales of four rows.
    const int r = blk * BLOCK_ROWS + (off < CODE_BYTES ? off / 32 : (off - CODE_BYTES) / 4);
    const bool keep = tile * TILE_ROWS + r < u.len;
    const int64_t at = static_cast<int64_t>(tile) * TILE_BLOCKS + (keep ? blk : 0);
#pragma unroll
    for (int kv = 0; kv < 2; ++kv)
      copy16_or_zero(dst + kv * HALF_BYTES + c * 16, u.base[kv] + at * p.cache[kv].sn + off, keep);
  }
}

// Sixteen bf16 features of a query row as they are in memory; zeros for a row that is not there.
struct RawQuery {
  uint4 lo, hi;
  __device__ __forceinline__ void load(const __nv_bfloat16* src, bool row) {
    lo = hi = make_uint4(0, 0, 0, 0);
    if (!row) return;
    lo = *reinterpret_cast<const uint4*>(src);
    hi = *reinterpret_cast<const uint4*>(src + 8);
  }
};

// A query row's features (16 of them) as half pairs, scaled by a power of two so that the row's largest element (over
// the four lanes t4) is in [2^14, 2^15). Returns the factor that turns products with them into exponents of 2.
__device__ __forceinline__ float scale_query(const RawQuery& raw, uint32_t (&qf)[8]) {
  float x[16], lo[8], hi[8], top = 0.0f;
  norm_rope::unpack8(raw.lo, lo);
  norm_rope::unpack8(raw.hi, hi);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = lo[i];
    x[i + 8] = hi[i];
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
  for (int i = 0; i < 8; ++i) qf[i] = pack_half2(x[2 * i] * up0 * up1, x[2 * i + 1] * up0 * up1);
  return 0.125f * 1.44269504088896340736f / up0 / up1;
}

// Scale bytes of rows first .. (to the end of their group of four) of K and V become zero: these rows are behind the
// last one and came with its group, so anything may stand there.
__device__ __forceinline__ void clear_tail(uint32_t ks, int first, int lane) {
  const int last = min((first + 3) & ~3, TILE_ROWS);
  for (int i = lane; i < (last - first) * 2 * GROUPS; i += 32) {
    const int r = first + i / (2 * GROUPS), j = i % (2 * GROUPS);
    sts_u8(ks + (j < GROUPS ? 0 : HALF_BYTES) + (r / BLOCK_ROWS) * BLOCK_BYTES + CODE_BYTES +
               (r % BLOCK_ROWS) * GROUPS + j % GROUPS, 0);
  }
  __syncwarp();
}

// V's A fragments of a block: values of tokens (t4, 4 + t4) and (8 + t4, 12 + t4) in half 0 and 1; features 8 g + 2 i
// at i, + 1 at 4 + i. The codes of two rows are interleaved, then converted and scaled.
__device__ __forceinline__ void value_fragments(uint32_t codes, uint32_t scales, uint32_t (&a)[2][8]) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const uint32_t w0 = lds_u32(codes + half * 8 * (HD / 2)), w1 = lds_u32(codes + (half * 8 + 4) * (HD / 2));
    const uint32_t even = (w0 & 0x0f0f0f0fu) | ((w1 << 4) & 0xf0f0f0f0u);
    const uint32_t odd = ((w0 >> 4) & 0x0f0f0f0fu) | (w1 & 0xf0f0f0f0u);
    uint32_t x[4], y[4];
    decode8(even, x);
    decode8(odd, y);
    // The scales of the two tokens as a half pair.
    const uint32_t from = scales + half * 8 * GROUPS;
    const uint32_t scale = (lds_u8(from) << 7) + (lds_u8(from + 4 * GROUPS) << 23);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[half][i] = mul_half2(x[i], scale);
      a[half][4 + i] = mul_half2(y[i], scale);
    }
  }
}

// A warp's query rows of one unit and the softmax over the tiles it has seen.
template <int NT, bool ONE>
struct Rows {
  static constexpr int COLS = 2;
  uint32_t qf[NT][8];          // Q as B fragments: query row n = g of each eight, features 16 t4 .. + 15
  float factor[NT][COLS];      // turns the products of query row 2 t4 + j into exponents of 2
  int hidden_rows[NT][COLS];   // the last rows of the cache that it does not see
  float acc[NT][4][4];         // O^T: features 8 g + 2 i (+ 1 in 2, 3), query rows 2 t4, 2 t4 + 1
  float mx[NT][COLS];          // running maximum, the same in all lanes of a column
  float ref[NT][COLS];         // exponent that weights are relative to: mx - RAISE
  float total[NT][COLS];       // weights, this lane's cached rows only

  struct Raw {
    RawQuery row[NT];
  };
  __device__ __forceinline__ Raw fetch(const Params& p, const Unit& u, int lane) const {
    constexpr int ROWS = 8 * NT;
    const int g = lane >> 2, t4 = lane & 3;
    const int rows = min(p.G * p.T - u.rt * ROWS, ROWS);
    Raw raw;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = n * 8 + g, gr = u.rt * ROWS + r;
      raw.row[n].load(p.q + u.b * p.q_sb + (u.hk * p.G + gr / p.T) * p.q_sh + (gr % p.T) * p.q_st + 16 * t4,
                      r < rows);
    }
    return raw;
  }

  __device__ __forceinline__ void begin(const Params& p, const Unit& u, const Raw& raw, int lane) {
    constexpr int ROWS = 8 * NT;
    const int t4 = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float f = scale_query(raw.row[n], qf[n]);
#pragma unroll
      for (int j = 0; j < COLS; ++j) {
        factor[n][j] = __shfl_sync(0xffffffffu, f, (2 * t4 + j) * 4);
        hidden_rows[n][j] = p.T - 1 - (u.rt * ROWS + n * 8 + 2 * t4 + j) % p.T;
        mx[n][j] = NEG_INF;
        ref[n][j] = total[n][j] = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[n][i][j] = 0.0f;
    }
  }

  // One tile in shared memory (K at ks, V behind it).
  __device__ __forceinline__ void tile(const Params& p, int len, int row0, uint32_t ks, int lane) {
    const int g = lane >> 2, t4 = lane & 3;
    const uint32_t vs = ks + HALF_BYTES;
    const bool masked = row0 + TILE_ROWS > len - (p.T - 1);
    uint32_t hidden = 0;
    const int hidden0 = max(row0, len - (p.T - 1));
    if (masked) {
      if (row0 + TILE_ROWS > len) clear_tail(ks, len - row0, lane);
      // A value that is not finite, in a row that some queries see and others do not, would reach them all as
      // 0 x NaN: its group counts as zero in the product, and as NaN for those that see it. hidden: such rows
      // (from hidden0) of this lane's group of features.
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
    const uint32_t kcodes = ks + kr * (HD / 2) + t4 * 8, kscales = ks + CODE_BYTES + kr * GROUPS + t4;
#pragma unroll
    for (int j = 0; j < TILE_BLOCKS; ++j) {
      uint32_t a[2][8];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint2 w = lds_u2(kcodes + j * BLOCK_BYTES + half * 8 * (HD / 2));
        const uint32_t scale = scale_pair(lds_u8(kscales + j * BLOCK_BYTES + half * 8 * GROUPS));
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
        mma_f16_first(s[j][n], a[0][0], a[1][0], a[0][1], a[1][1], qf[n][0], qf[n][1]);
#pragma unroll
        for (int k = 1; k < 4; ++k)
          mma_f16(s[j][n], a[0][2 * k], a[1][2 * k], a[0][2 * k + 1], a[1][2 * k + 1], qf[n][2 * k],
                  qf[n][2 * k + 1]);
      }
    }
    // ---- masks, the running maximum
    if (masked) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < TILE_BLOCKS; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (row0 + j * BLOCK_ROWS + kr + 8 * (i >> 1) >= len - hidden_rows[n][i & 1])
              s[j][n][i] = NEG_INF;
    }
    bool over = false;
    float top[NT][COLS];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < COLS; ++c) {
        float m = fmaxf(s[0][n][c], s[0][n][2 + c]);
#pragma unroll
        for (int j = 1; j < TILE_BLOCKS; ++j) m = fmax3(m, s[j][n][c], s[j][n][2 + c]);
        top[n][c] = m * factor[n][c];   // a factor is positive
        over = over || top[n][c] > mx[n][c] + SLACK;
      }
    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
          float m = fmaxf(top[n][c], mx[n][c]);
#pragma unroll
          for (int d = 4; d < 32; d *= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
          const float old = ref[n][c];
          const bool empty = mx[n][c] == NEG_INF;
          mx[n][c] = m;
          ref[n][c] = m == NEG_INF ? 0.0f : m - RAISE;
          const float f = empty ? 1.0f : ex2_approx(old - ref[n][c]);   // empty: the sums are zero, or NaN
          total[n][c] *= f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            acc[n][i][c] *= f;
            acc[n][i][2 + c] *= f;
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
          e[i] = ex2_approx(fmaf(s[j][n][i], factor[n][i & 1], -ref[n][i & 1]));
          total[n][i & 1] += e[i];
        }
        pf[j][n][0] = transpose8x8(pack_half2(e[0], e[1]));
        pf[j][n][1] = transpose8x8(pack_half2(e[2], e[3]));
      }
    // ---- O^T += V^T P^T
    const uint32_t vcodes = vs + t4 * (HD / 2) + g * 4, vscales = vs + CODE_BYTES + t4 * GROUPS + (g >> 1);
#pragma unroll
    for (int j = 0; j < TILE_BLOCKS; ++j) {
      uint32_t a[2][8];
      value_fragments(vcodes + j * BLOCK_BYTES, vscales + j * BLOCK_BYTES, a);
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
        for (int c = 0; c < COLS; ++c) {
          // Bits of the rows that this query sees.
          const int seen = len - hidden_rows[n][c] - hidden0;
          if (seen > 0 && (hidden & ((2u << min(seen - 1, 30)) - 1u)) != 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[n][i][c] = acc[n][i][2 + c] = __uint_as_float(0x7fffffffu);
          }
        }
    }
  }

  // The warp's record: [query row][feature], reference exponent, total.
  __device__ __forceinline__ void end(float (*rec)[REC], int rows, int lane) {
    const int g = lane >> 2, t4 = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < COLS; ++c) {
        float sum = total[n][c];
#pragma unroll
        for (int d = 4; d < 32; d *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        const int r = n * 8 + 2 * t4 + c;
        if (r >= rows) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<float2*>(rec[r] + 8 * g + 2 * i) = make_float2(acc[n][i][c], acc[n][i][2 + c]);
        // Weightless but not empty: NaN scores leave the maximum alone.
        if (g == 0)
          *reinterpret_cast<float2*>(rec[r] + HD) =
              make_float2(mx[n][c] == NEG_INF && sum == 0.0f ? NEG_INF : ref[n][c], sum);
      }
  }
};

// A single query row: the products' eight columns stand for the scale groups (two columns each), so that the codes need
// no scaling.
//   S: column n of B is q where a lane's features belong to group n % 4 and zero elsewhere; a row's four sums times
//      their scales are added in FP32.
//   O: as with more rows, all columns alike. (Scales in B, p x scale in half precision, would spare the multiplications
//   of V too, but leave half precision's range: rows behind a heavy one, or with small values, were lost.)
// 16 multiplications a block of 16 rows less (64 sequences x 12 heads, 1024-8192 rows: 54.6 -> 49.7 us).
template <>
struct Rows<1, true> {
  uint32_t qf[8];
  float factor, mx, ref, total;
  float acc[4][4];   // features 8 g + 2 i (+ 1 in 2, 3)

  __device__ __forceinline__ RawQuery fetch(const Params& p, const Unit& u, int lane) const {
    RawQuery raw;
    raw.load(p.q + u.b * p.q_sb + u.hk * p.q_sh + 16 * (lane & 3), true);
    return raw;
  }

  __device__ __forceinline__ void begin(const Params&, const Unit&, const RawQuery& raw, int lane) {
    const int g = lane >> 2, t4 = lane & 3;
    factor = scale_query(raw, qf);
    if ((g & 3) != t4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) qf[i] = 0;
    }
    mx = NEG_INF;
    ref = total = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
  }

  __device__ __forceinline__ void tile(const Params&, int len, int row0, uint32_t ks, int lane) {
    const int g = lane >> 2, t4 = lane & 3;
    const uint32_t vs = ks + HALF_BYTES;
    const bool tail = row0 + TILE_ROWS > len;
    if (tail) clear_tail(ks, len - row0, lane);
    // ---- scores of rows (g >> 1) + 4 (g & 1), and 8 more, of each block, in all four lanes t4
    float s[TILE_BLOCKS][2];
    const int kr = (g >> 1) + 4 * (g & 1);
    const uint32_t kcodes = ks + kr * (HD / 2) + t4 * 8, kscales = ks + CODE_BYTES + kr * GROUPS + 2 * (t4 & 1);
#pragma unroll
    for (int j = 0; j < TILE_BLOCKS; ++j) {
      uint32_t a[2][8];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint2 w = lds_u2(kcodes + j * BLOCK_BYTES + half * 8 * (HD / 2));
        uint32_t x[4], y[4];
        decode8(w.x, x);
        decode8(w.y, y);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          a[half][i] = x[i];
          a[half][4 + i] = y[i];
        }
      }
      float c[4];
      mma_f16_first(c, a[0][0], a[1][0], a[0][1], a[1][1], qf[0], qf[1]);
#pragma unroll
      for (int k = 1; k < 4; ++k)
        mma_f16(c, a[0][2 * k], a[1][2 * k], a[0][2 * k + 1], a[1][2 * k + 1], qf[2 * k], qf[2 * k + 1]);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        // Two scale bytes as halves, then floats: a NaN stays one (as a float's upper bits its byte would be a number).
        const uint32_t bytes = lds_u16(kscales + j * BLOCK_BYTES + half * 8 * GROUPS);
        const uint32_t pair = __byte_perm(bytes, 0, 0x4140) << 7;
        const float2 scale = __half22float2(*reinterpret_cast<const __half2*>(&pair));
        const float y = fmaf(c[2 * half], scale.x, c[2 * half + 1] * scale.y);
        s[j][half] = y + __shfl_xor_sync(0xffffffffu, y, 1);
      }
    }
    if (tail) {
#pragma unroll
      for (int j = 0; j < TILE_BLOCKS; ++j)
#pragma unroll
        for (int half = 0; half < 2; ++half)
          if (row0 + j * BLOCK_ROWS + kr + 8 * half >= len) s[j][half] = NEG_INF;
    }
    float top = fmaxf(s[0][0], s[0][1]);
#pragma unroll
    for (int j = 1; j < TILE_BLOCKS; ++j) top = fmax3(top, s[j][0], s[j][1]);
    top *= factor;
    if (__any_sync(0xffffffffu, top > mx + SLACK)) {
      float m = fmaxf(top, mx);
#pragma unroll
      for (int d = 4; d < 32; d *= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
      const float old = ref;
      const bool empty = mx == NEG_INF;
      mx = m;
      ref = m == NEG_INF ? 0.0f : m - RAISE;
      const float f = empty ? 1.0f : ex2_approx(old - ref);   // empty: the sums are zero, or NaN
      total *= f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] *= f;
    }
    uint32_t pf[TILE_BLOCKS][2];
#pragma unroll
    for (int j = 0; j < TILE_BLOCKS; ++j)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const float e = ex2_approx(fmaf(s[j][half], factor, -ref));
        total += e;
        pf[j][half] = transpose8x8(pack_half2(e, e));
      }
    const uint32_t vcodes = vs + t4 * (HD / 2) + g * 4, vscales = vs + CODE_BYTES + t4 * GROUPS + (g >> 1);
#pragma unroll
    for (int j = 0; j < TILE_BLOCKS; ++j) {
      uint32_t a[2][8];
      value_fragments(vcodes + j * BLOCK_BYTES, vscales + j * BLOCK_BYTES, a);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        mma_f16(acc[i], a[0][i], a[0][4 + i], a[1][i], a[1][4 + i], pf[j][0], pf[j][1]);
    }
  }

  __device__ __forceinline__ void end(float (*rec)[REC], int, int lane) {
    const int g = lane >> 2, t4 = lane & 3;
    float sum = total;
#pragma unroll
    for (int d = 4; d < 32; d *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (t4 == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<float2*>(rec[0] + 8 * g + 2 * i) = make_float2(acc[i][0], acc[i][2]);
    }
    if (lane == 0)
      *reinterpret_cast<float2*>(rec[0] + HD) = make_float2(mx == NEG_INF && sum == 0.0f ? NEG_INF : ref, sum);
  }
};

// Weight of a part with reference exponent e against the common one, 0 for an empty part.
__device__ __forceinline__ float part_weight(float e, float ref) {
  return e == NEG_INF ? 0.0f : ex2_approx(e - ref);
}

// Sums of several parts of a query row: this lane's two features, the reference exponent, the total weight.
struct Sum {
  float e = NEG_INF, l = 0.0f, v0 = 0.0f, v1 = 0.0f;

  // Up to N records from rec on, `step` floats apart, loaded together: one maximum, then all weights side by side.
  template <int N>
  __device__ __forceinline__ void add(const float* rec, int64_t step, int count, int lane) {
    float2 el[N], v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float* at = rec + (j < count ? j * step : 0);
      el[j] = *reinterpret_cast<const float2*>(at + HD);
      v[j] = *reinterpret_cast<const float2*>(at + 2 * lane);
    }
    float top = e;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (j >= count) el[j].x = NEG_INF;
      top = fmaxf(top, el[j].x);
    }
    const float f = part_weight(e, top);
    e = top;
    l *= f;
    v0 *= f;
    v1 *= f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float h = part_weight(el[j].x, top);
      l += j < count ? el[j].y * h : 0.0f;    // (a part that is not counted may hold anything)
      v0 += j < count ? v[j].x * h : 0.0f;
      v1 += j < count ? v[j].y * h : 0.0f;
    }
  }
  __device__ __forceinline__ void store(float* rec, int lane) const {
    *reinterpret_cast<float2*>(rec + 2 * lane) = make_float2(v0, v1);
    if (lane == 0) *reinterpret_cast<float2*>(rec + HD) = make_float2(e, l);
  }
  // O and LSE of the row.
  __device__ __forceinline__ void finish(const Params& p, int64_t row, int lane) const {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    *reinterpret_cast<uint32_t*>(p.o + row * HD + 2 * lane) = pack_bf16x2(v0 * inv, v1 * inv);
    if (p.lse != nullptr && lane == 0) p.lse[row] = l == 0.0f ? NEG_INF : (e + __log2f(l)) * LN2;
  }
};

// ------------------------------------------------------------------------------- cluster kernel

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

// One cluster (or several: parts) shares the tiles of a unit.
template <int NT, bool ONE>
__global__ void __launch_bounds__(THREADS, NT == 1 ? MIN_CTAS : 3)
    attention_kernel(const __grid_constant__ Params p) {
  constexpr int ROWS = 8 * NT;
  extern __shared__ uint8_t smem_raw[];
  Smem<NT>& sm = *reinterpret_cast<Smem<NT>*>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(blockIdx.x) % p.cluster;
  const int pc = static_cast<int>(blockIdx.x) / p.cluster;      // unit * parts + part
  const int part = pc % p.parts, unit = pc / p.parts;
  const int rt = unit % p.row_tiles, bh = unit / p.row_tiles;
  const int rows = min(p.G * p.T - rt * ROWS, ROWS);
  const int workers = WARPS * p.cluster * p.parts;
  const int worker = (part * p.cluster + rank) * WARPS + warp;
  // Arrived at before the others' shared memory is written: a CTA that has not started has none.
  if (p.cluster > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  wait_for_previous_kernel();

  const bool dense = p.cache[0].sn == BLOCK_BYTES && p.cache[1].sn == BLOCK_BYTES;
  Unit u;
  u.set(p, bh / p.Hkv, bh % p.Hkv, rt, visible_rows(p, bh / p.Hkv));
  const uint32_t ring = smem_u32(sm.warp[warp].ring);
  Rows<NT, ONE> q;
  const auto raw = q.fetch(p, u, lane);
  int next = worker;
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) {
    if (next < u.tiles) load_tile(p, u, next, ring + s * STAGE_BYTES, lane, dense);
    copy_commit();
    next += workers;
  }
  q.begin(p, u, raw, lane);
  int stage = 0;
#pragma unroll 1
  for (int tile = worker; tile < u.tiles; tile += workers) {
    copy_wait<STAGES - 2>();
    __syncwarp();
    // Into the stage of the step before, which every lane has left.
    if (next < u.tiles)
      load_tile(p, u, next, ring + (stage == 0 ? STAGES - 1 : stage - 1) * STAGE_BYTES, lane, dense);
    copy_commit();
    next += workers;
    q.tile(p, u.len, tile * TILE_ROWS, ring + stage * STAGE_BYTES, lane);
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
  copy_wait<0>();
  __syncwarp();
  q.end(sm.warp[warp].own, ROWS, lane);
  __syncthreads();
  // ---- the CTA's record, at the cluster's CTA that finishes the row: row r at rank r % cluster
  const int64_t row0 = static_cast<int64_t>(bh) * p.G * p.T + rt * ROWS;
  if (p.cluster > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  for (int r = warp; r < rows; r += WARPS) {
    Sum sum;
    sum.add<WARPS>(sm.warp[0].own[r], sizeof(sm.warp[0]) / sizeof(float), WARPS, lane);
    if (p.cluster > 1) {
      const uint32_t dst = map_to_rank(smem_u32(sm.from[r / p.cluster * p.cluster + rank]),
                                       static_cast<uint32_t>(r % p.cluster));
      st_cluster_f32x2(dst + lane * 8, sum.v0, sum.v1);
      if (lane == 0) st_cluster_f32x2(dst + HD * 4, sum.e, sum.l);
    } else if (p.parts > 1) {
      sum.store(p.records + (static_cast<int64_t>(pc) * ROWS + r) * REC, lane);
    } else {
      sum.finish(p, row0 + r, lane);
    }
  }
  if (p.cluster == 1) return;
  __syncwarp();
  cluster_sync();
  for (int r = rank + p.cluster * warp; r < rows; r += p.cluster * WARPS) {
    Sum sum;
    sum.add<MAX_CLUSTER>(sm.from[r / p.cluster * p.cluster], REC, p.cluster, lane);
    if (p.parts > 1)
      sum.store(p.records + (static_cast<int64_t>(pc) * ROWS + r) * REC, lane);
    else
      sum.finish(p, row0 + r, lane);
  }
}

// ------------------------------------------------------------------------------- merging records

constexpr int COMBINE_WARPS = 8;
constexpr int COMBINE_LOADS = 4;   // records of a warp in flight

// Merges the parts' records: one CTA a row, each warp every eighth part.
__global__ void __launch_bounds__(COMBINE_WARPS * 32)
    combine_kernel(const __grid_constant__ Params p, int tile_rows) {
  __shared__ float rec[COMBINE_WARPS][REC];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_head = p.G * p.T;
  const int bh = static_cast<int>(blockIdx.x) / per_head, gr = static_cast<int>(blockIdx.x) % per_head;
  const int64_t unit = static_cast<int64_t>(bh) * p.row_tiles + gr / tile_rows;
  wait_for_previous_kernel();
  const float* src = p.records + (unit * p.parts * tile_rows + gr % tile_rows) * REC;
  Sum sum;
  const int64_t step = static_cast<int64_t>(tile_rows) * REC * COMBINE_WARPS;
  src += warp * (step / COMBINE_WARPS);
  for (int c = warp; c < p.parts; c += COMBINE_WARPS * COMBINE_LOADS, src += COMBINE_LOADS * step)
    sum.add<COMBINE_LOADS>(src, step, (p.parts - c + COMBINE_WARPS - 1) / COMBINE_WARPS, lane);
  sum.store(rec[warp], lane);
  __syncthreads();
  if (warp != 0) return;
  Sum all;
  all.add<COMBINE_WARPS>(rec[0], REC, COMBINE_WARPS, lane);
  all.finish(p, blockIdx.x, lane);
}

// ------------------------------------------------------------------------------- flat kernel

// Many units: the tiles of all of them stand in one row, which is cut into equal shares, one for each warp of a grid that
// fills the SMs once, whatever the lengths. One CTA of 12 or 16 warps to an SM: with four CTAs of four the warps of
// the older CTAs ran ahead and the last one took 47 us where the mean was 38. A share's tiles of a unit end in
// a record at slot worker + unit (neither decreases along the row, so no two have the same), and
// flat_combine_kernel merges a unit's records in their order.
template <int NT>
struct Flat {
  static constexpr int WARPS = NT == 1 ? 16 : 12;
  static constexpr size_t SMEM = static_cast<size_t>(WARPS) * STAGES * STAGE_BYTES;
};

__device__ __forceinline__ int unit_tiles(const Params& p, int b) {
  return (visible_rows(p, b) + TILE_ROWS - 1) / TILE_ROWS;
}

// The cut of `total` tiles into shares: none is empty, and they differ by one tile.
struct Shares {
  int workers, each, more;   // the first `more` shares have each + 1 tiles

  __device__ __forceinline__ void set(int total, int most) {
    workers = max(1, min(most, total));
    each = total / workers;
    more = total - each * workers;
  }
  __device__ __forceinline__ int first(int worker) const { return each * worker + min(worker, more); }
  __device__ __forceinline__ int owner(int tile) const {
    const int longer = more * (each + 1);
    return tile < longer ? tile / (each + 1) : more + (tile - longer) / each;
  }
};

// Sum of v over the lanes up to this one.
__device__ __forceinline__ int lanes_up_to(int v, int lane) {
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int x = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += x;
  }
  return v;
}

// A place in the row of tiles.
struct Cursor {
  Unit u;
  int tile;

  // To the next tile; there is one.
  __device__ __forceinline__ void step(const Params& p) {
    if (++tile < u.tiles) return;
    tile = 0;
    int rt = u.rt + 1, hk = u.hk, b = u.b, len = u.len;
    if (rt == p.row_tiles) {
      rt = 0;
      if (++hk == p.Hkv) {
        hk = 0;
        do {
          len = visible_rows(p, ++b);
        } while (len == 0);
      }
    }
    u.set(p, b, hk, rt, len);
  }
  // To tile `at` behind the first one of sequence b0.
  __device__ __forceinline__ void seek(const Params& p, int b0, int at, int lane) {
    const int heads = p.Hkv * p.row_tiles;
    for (;; b0 += 32) {
      const int n = b0 + lane < p.B ? unit_tiles(p, b0 + lane) * heads : 0;
      const int up = lanes_up_to(n, lane);   // tiles up to this lane's sequence
      const unsigned here = __ballot_sync(0xffffffffu, up > at);
      if (here == 0 && b0 + 32 < p.B) {
        at -= __shfl_sync(0xffffffffu, up, 31);
        continue;
      }
      const int l = here != 0 ? __ffs(static_cast<int>(here)) - 1 : 0;
      at -= __shfl_sync(0xffffffffu, up - n, l);
      const int b = b0 + l, tiles = max(1, unit_tiles(p, b)), in = at / tiles;
      tile = at - in * tiles;
      u.set(p, b, in / p.row_tiles, in % p.row_tiles, visible_rows(p, b));
      return;
    }
  }
};

// The register limits leave room for a merging CTA beside this kernel's (launched early, it waits for the records).
template <int NT, bool ONE>
__global__ void __maxnreg__(NT == 1 ? 112 : 152)
    flat_kernel(const __grid_constant__ Params p) {
  constexpr int ROWS = 8 * NT, W = Flat<NT>::WARPS;
  extern __shared__ uint8_t smem_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ring = smem_u32(smem_raw) + warp * STAGES * STAGE_BYTES;
  const int worker = static_cast<int>(blockIdx.x) * W + warp;
  wait_for_previous_kernel();
  // The merge's launch runs under this kernel.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const bool dense = p.cache[0].sn == BLOCK_BYTES && p.cache[1].sn == BLOCK_BYTES;
  // Each warp counts the tiles of a range of sequences; the ranges' sums tell where this warp's share begins. (A range for
  // each lane made 4096 sequences take 32 us longer: its loads lie apart.)
  __shared__ int range_tiles[W];
  const int range = (p.B + W * 32 - 1) / (W * 32) * 32;
  int mine = 0;
#pragma unroll 4
  for (int b = warp * range + lane; b < min(p.B, (warp + 1) * range); b += 32) mine += unit_tiles(p, b);
  mine = __reduce_add_sync(0xffffffffu, mine) * p.Hkv * p.row_tiles;
  if (lane == 0) range_tiles[warp] = mine;
  __syncthreads();
  const int up = lanes_up_to(lane < W ? range_tiles[lane] : 0, lane);
  Shares shares;
  shares.set(__shfl_sync(0xffffffffu, up, 31), static_cast<int>(gridDim.x) * W);
  if (worker >= shares.workers || shares.each == 0) return;
  const int first = shares.first(worker), count = shares.first(worker + 1) - first;
  const int l = __ffs(static_cast<int>(__ballot_sync(0xffffffffu, up > first))) - 1;
  Cursor now, ahead;
  now.seek(p, l * range, first - (l > 0 ? __shfl_sync(0xffffffffu, up, l - 1) : 0), lane);
  ahead = now;
  Rows<NT, ONE> q;
  auto raw = q.fetch(p, now.u, lane);
  int loaded = 0;
  auto load_next = [&](int stage) {
    if (loaded < count) {
      load_tile(p, ahead.u, ahead.tile, ring + stage * STAGE_BYTES, lane, dense);
      if (++loaded < count) ahead.step(p);
    }
    copy_commit();
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) load_next(s);
  q.begin(p, now.u, raw, lane);
  int stage = 0;
#pragma unroll 1
  for (int i = 1; i <= count; ++i) {
    copy_wait<STAGES - 2>();
    __syncwarp();
    // Into the stage of the step before, which every lane has left.
    load_next(stage == 0 ? STAGES - 1 : stage - 1);
    q.tile(p, now.u.len, now.tile * TILE_ROWS, ring + stage * STAGE_BYTES, lane);
    stage = stage + 1 == STAGES ? 0 : stage + 1;
    if (i < count && now.tile + 1 < now.u.tiles) {
      ++now.tile;
      continue;
    }
    const int unit = (now.u.b * p.Hkv + now.u.hk) * p.row_tiles + now.u.rt;
    q.end(reinterpret_cast<float(*)[REC]>(p.records) + (static_cast<int64_t>(worker) + unit) * ROWS,
          min(p.G * p.T - now.u.rt * ROWS, ROWS), lane);
    if (lane == 0 && now.tile + 1 == now.u.tiles) {
      const int from = shares.owner(first + i - 1 - now.tile);
      p.parts_of[unit] = make_int2(from, worker - from + 1);
    }
    if (i == count) break;
    now.step(p);
    raw = q.fetch(p, now.u, lane);
    q.begin(p, now.u, raw, lane);
  }
}

constexpr int FLAT_COMBINE_WARPS = 4;
constexpr int FLAT_COMBINE_LOADS = 4;   // records in flight

// One warp a query row: the records of the shares that hold tiles of its unit.
__global__ void __launch_bounds__(FLAT_COMBINE_WARPS * 32, 8)
    flat_combine_kernel(const __grid_constant__ Params p, int tile_rows) {
  const int lane = threadIdx.x & 31;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * FLAT_COMBINE_WARPS + (threadIdx.x >> 5);
  const int per_head = p.G * p.T;
  const bool valid = at < static_cast<int64_t>(p.B) * p.Hkv * per_head;
  const int bh = valid ? static_cast<int>(at / per_head) : 0, gr = valid ? static_cast<int>(at % per_head) : 0;
  const int unit = bh * p.row_tiles + gr / tile_rows, b = bh / p.Hkv;
  wait_for_previous_kernel();
  if (!valid) return;   // whole warps
  const int len = visible_rows(p, b);
  const int2 parts = p.parts_of[unit];   // (not written for a unit without tiles)
  const int w0 = len > 0 ? parts.x : 0, count = len > 0 ? parts.y : 0;
  const int64_t step = static_cast<int64_t>(tile_rows) * REC;
  const float* src = p.records + (static_cast<int64_t>(w0) + unit) * step + gr % tile_rows * REC;
  Sum sum;
  for (int i = 0; i < count; i += FLAT_COMBINE_LOADS, src += FLAT_COMBINE_LOADS * step)
    sum.add<FLAT_COMBINE_LOADS>(src, step, count - i, lane);
  sum.finish(p, at, lane);
}

}  // namespace attn
}  // namespace cache4
}  // namespace tt
