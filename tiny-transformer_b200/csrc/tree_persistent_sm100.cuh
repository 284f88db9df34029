// Tree attention as one persistent kernel on the fifth-generation tensor cores (the operator and
// its rules: tree_attention_sm100.cuh).
//
// Split. A unit is one (batch, K/V head, row tile of up to 128 stacked query rows); its tiles are
// the tree's key tiles, then the cache's, 128 keys each. All units' tiles form one flat list in
// (batch, unit, tile) order, each unit with UNIT_COST tiles' worth of cost in front (its epilogue
// and first loads), and CTA i of the grid (one per SM) takes the i-th equal part of the cost, found
// from the lengths on the device: uneven lengths and few long sequences load every SM alike, and a
// CTA has at most two units that it shares with others (its first and its last). Those leave an FP32 record per row (O, m, l) in the workspace, which tree_combine_kernel merges; units
// that lie in one CTA are written directly.
//
// Work of one CTA. S (128 x 128) = Q K^T and O (128 x 64) += P V are tcgen05.mma with M = 128 rows
// in TMEM. Trees have far fewer than 128 rows (the kernel is bound by reading the cache, the
// products of a full tile take about a third of that time), so for at most 64 or 32 rows the tile
// holds DUP = 2 or 4 copies of Q, and copy c works on the c-th 128 / DUP keys of every tile only:
// its other P entries are zero, its running max and sums are its own, and the copies merge at the
// end of the unit like the CTAs do. So all four softmax warps have work whatever the row count, a
// thread takes 128 / DUP exponentials a tile, and the tensor work does not change. All exponentials
// are MUFU ones: the FMA-pipe polynomial of the prefill kernel (1e-4) shows in the LSE, and the
// softmax is not the bound here. P is rounded to BF16 (see tree_attention_sm100.cuh), the sums take it
// before. O is rescaled only when a row's max grows by more than 2^8.
//
// Roles: two softmax warpgroups (warps 0-3 and 4-7, thread = TMEM lane) take the tiles alternately,
// each with score, P and O columns, a running max and a sum of its own (they merge like the
// copies): one warpgroup alone needed about 1400 cycles a tile (TMEM reads, 64 exponentials and
// the hand-overs in series), as long as the memory needs to deliver it. Warp 8 is the TMA producer
// (rings of K and V tiles of their own, so that K is released once its scores are computed), warp
// 9 issues S as soon as the scores two tiles back have been read, warp 10 issues P.V (an issuing
// thread blocks while the tensor core works, so one thread for both made a tile cost the sum of
// their times), warp 11 loads Q and builds the ancestor masks of the next unit. TMEM (512
// columns): per warpgroup S (128), P (64), O (64). Every wait is bounded.
//
// Measured (B200): 68 us, 3.9 TB/s and 237 TFLOP/s, for 32 sequences x 12 heads of 1024-4096 cached
// rows and 64 nodes: a tile takes about 1250 cycles of a CTA, what the memory needs to deliver it,
// but the start (6000 cycles), 3.6 units' epilogues a CTA (4000 each, in which the ring of four
// tiles fills up) and the merge kernel (6 us) come on top. 31 us for 3 sequences x 4 K/V heads of 9000-
// 20001 rows, 37 nodes and 3 query heads each (9 tiles a CTA of 1700 cycles: a thread
// has 128 exponentials a tile, 1024 cycles of the MUFU units, and the kernel with one copy of Q, alone of
// the three, spills 144 bytes; start, tiles, epilogues and merge add up to 21 of the 31 us, the rest is
// not accounted for). Tried: one softmax warpgroup 96 us; scores held 64 at a time with
// spills, with and without handing registers over (setmaxnreg) 94-122; equal tiles instead of equal
// cost per CTA 74; S and P.V from one thread 115.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cstdint>
#include <type_traits>

#include "sm100_ptx.cuh"
#include "tree_attention_sm100.cuh"

namespace tt {
namespace tree {
namespace persist {

constexpr int BM = 128;
constexpr int GROUPS = 2;                         // softmax warpgroups
constexpr int SOFTMAX_WARPS = 4 * GROUPS;
constexpr int LOAD_WARP = SOFTMAX_WARPS;
constexpr int S_WARP = SOFTMAX_WARPS + 1;
constexpr int PV_WARP = SOFTMAX_WARPS + 2;
constexpr int THREADS = (SOFTMAX_WARPS + 4) * 32;
constexpr int K_STAGES = 4;
constexpr int V_STAGES = 4;
constexpr uint32_t S_COL = 0, P_COL = 256, O_COL = 384, TMEM_COLS = 512;
constexpr float RESCALE_THRESHOLD = 8.0f;
constexpr unsigned UNIT_COST = 3;                 // a unit's fixed cost, in tiles
constexpr int MERGE_COLS = 32;                    // O columns merged at a time
constexpr uint32_t MERGE_BYTES = (MERGE_COLS + 4) * 4;
constexpr int COMBINE_ROWS = 8;                   // rows per combine block
constexpr int COMBINE_SHARES = 2;                 // threads that share a row's records
constexpr int COMBINE_THREADS = COMBINE_ROWS * 8 * COMBINE_SHARES;

// Where a CTA's part of the flat list starts (all counts fit 32 bits: the host checks).
struct Start {
  int b, unit, tile;
  int count;  // tiles of the CTA
  int tiles;  // of the unit
  int pad[3];
};

struct Params {
  tree::Params t;
  int rows;                     // query rows of a unit's tile (the last tile may have fewer)
  int units;                    // units per batch row: Hkv * row_tiles
  int tree_tiles;
  bool whole;                   // parts begin and end at units: nothing to merge
  Start* starts;                // [grid]: workspace
  float* records;               // [grid][2][rows][REC]: workspace; 0: unit begun by another CTA
};

// A unit as the Q warp publishes it with Q, so that the softmax warps divide nothing.
struct Unit {
  int b, h;         // batch row, K/V head
  int row0, rows;   // first query row, query rows
  int len;          // cached rows
};

struct alignas(1024) Smem {
  uint8_t q[2][TILE_BYTES];
  uint8_t k[K_STAGES][TILE_BYTES];
  uint8_t v[V_STAGES][TILE_BYTES];
  float merge[GROUPS * BM][MERGE_COLS + 4];  // one column block of every thread's weighted O
  float ml[GROUPS * BM][2];                  // every thread's max and sum
  Unit unit[2];
  uint32_t mask[2][MAX_NODES][MASK_WORDS];
  int32_t jump[MAX_NODES];
  uint32_t bad[2][MASK_WORDS];  // nodes whose V row holds an infinity or a NaN
  int any_bad[2];
  uint64_t k_full[K_STAGES], k_empty[K_STAGES], v_full[V_STAGES], v_empty[V_STAGES];
  uint64_t q_full[2], q_free[2];
  uint64_t s_full[GROUPS], s_read[GROUPS], p_ready[GROUPS], pv_done[GROUPS], drain[2];
  Start start;
  uint32_t tmem_base;
  volatile int abort;
};
constexpr size_t kSmemBytes = sizeof(Smem);
static_assert(kSmemBytes <= 227 * 1024, "shared memory");

__device__ __forceinline__ int tiles_of(const Params& p, int b) {
  return p.tree_tiles + (valid_len(p.t.lens, p.t.C, b) + KEYS - 1) / KEYS;
}

// One warp: the CTA's part [total * i / grid, total * (i + 1) / grid) of the list, in cost. A cost
// position inside a unit is tile max(0, position - UNIT_COST): a part that ends in a unit's fixed
// cost ends before the unit, so parts may be empty, but not those that begin inside a unit. With
// p.whole a position moves to the nearer end of its unit.
__device__ __forceinline__ Start find_start(const Params& p, unsigned cta, unsigned grid, int lane) {
  // The lengths of the first 32 batch rows stay in a register, later ones are read again (L1).
  const unsigned tiles0 = lane < p.t.B ? tiles_of(p, lane) : 0;
  unsigned total = lane < p.t.B ? tiles0 + UNIT_COST : 0;
  for (int b = lane + 32; b < p.t.B; b += 32) total += tiles_of(p, b) + UNIT_COST;
  total = __reduce_add_sync(0xffffffffu, total) * p.units;
  if (total < grid) {
    if (cta >= total) return Start{};
    grid = total;
  }
  const unsigned each = total / grid, rest = total - each * grid;
  const unsigned from = each * cta + rest * cta / grid;
  const unsigned to = each * (cta + 1) + rest * (cta + 1) / grid;
  Start s{};
  unsigned before = 0, tiles_before = 0;  // cost, and tiles, of the batch rows so far
  unsigned first = 0;                     // tiles in front of the part
  bool found = false;
  for (int base = 0; base < p.t.B; base += 32) {
    const int b = base + lane;
    const unsigned tiles = base == 0 ? tiles0 : b < p.t.B ? tiles_of(p, b) : 0;
    const unsigned cost = b < p.t.B ? (tiles + UNIT_COST) * p.units : 0;
    unsigned run = cost;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const unsigned y = __shfl_up_sync(0xffffffffu, run, off);
      if (lane >= off) run += y;
    }
    // The row that holds a position, its unit and tile: the same steps for both ends.
    for (int end = found ? 1 : 0; end < 2; ++end) {
      const unsigned at = end == 0 ? from : to;
      const unsigned hit = __ballot_sync(0xffffffffu, before + run > at);
      if (hit == 0) break;
      const int l = __ffs(hit) - 1;
      const unsigned t = __shfl_sync(0xffffffffu, tiles, l);
      const unsigned in_b = at - before - __shfl_sync(0xffffffffu, run - cost, l);
      unsigned unit = in_b / (t + UNIT_COST);
      const unsigned in_unit = in_b - unit * (t + UNIT_COST);
      unsigned tile = in_unit > UNIT_COST ? in_unit - UNIT_COST : 0;
      if (p.whole) {
        tile = 0;
        if (2 * in_unit >= t + UNIT_COST) ++unit;  // p.units: the next row's first, see below
      }
      // Tiles before this row: its cost without the fixed parts.
      const unsigned row_tiles_before =
          tiles_before + __shfl_sync(0xffffffffu, run - cost, l) - UNIT_COST * p.units * l;
      const unsigned flat = row_tiles_before + unit * t + tile;
      if (end == 0) {
        found = true;
        first = flat;
        s.b = base + l;
        s.unit = static_cast<int>(unit);
        s.tile = static_cast<int>(tile);
        s.tiles = static_cast<int>(t);
        if (s.unit == p.units) {
          s.unit = 0;
          ++s.b;
          s.tiles = s.b < p.t.B ? tiles_of(p, s.b) : 0;
        }
      } else {
        s.count = static_cast<int>(flat - first);
        return s;
      }
    }
    const unsigned rows = min(32, p.t.B - base);
    const unsigned sum = __shfl_sync(0xffffffffu, run, 31);
    before += sum;
    tiles_before += sum - UNIT_COST * p.units * rows;
  }
  s.count = static_cast<int>(tiles_before - first);  // the part ends with the list
  return s;
}

// The CTA's units in order: [t0, t0 + n) of unit `unit` of batch row b.
struct Walk {
  int b, unit, t0, n, tiles, seg, left;
  int next_len;  // requested one batch row ahead
  __device__ __forceinline__ void begin(const Params& p, const Start& s) {
    b = s.b;
    unit = s.unit;
    t0 = s.tile;
    seg = 0;
    left = s.count;
    tiles = s.tiles;
    n = min(left, tiles - t0);
    prefetch(p);
  }
  __device__ __forceinline__ void prefetch(const Params& p) {
    next_len = p.t.lens != nullptr && b + 1 < p.t.B ? p.t.lens[b + 1] : p.t.C;
  }
  __device__ __forceinline__ void next(const Params& p) {
    left -= n;
    t0 = 0;
    ++seg;
    if (++unit == p.units) {
      unit = 0;
      ++b;
      tiles = p.tree_tiles + (min(max(next_len, 0), p.t.C) + KEYS - 1) / KEYS;
      prefetch(p);
    }
    n = min(left, tiles);
  }
};

// Maximum that is NaN when an argument is: a row with a NaN score is NaN as a whole.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Maximum of 32 scores by three-input maxima.
__device__ __forceinline__ float max32(const float (&x)[32]) {
  float a[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    a[i] = max3_nan(x[i], x[i + 8], x[i + 16]);
    a[i] = max3_nan(a[i], x[i + 24], x[i + 24]);
  }
  return max3_nan(max3_nan(a[0], a[1], a[2]), max3_nan(a[3], a[4], a[5]),
                  max3_nan(a[6], a[7], a[7]));
}

// P = exp2(x * sl2 - m) of 32 scores as bf16x2 to 16 columns at t_p; adds to the FP32 row sums.
__device__ __forceinline__ void exp_store32(const float (&x)[32], uint64_t sc2, uint64_t nm2,
                                            uint32_t t_p, uint64_t (&acc)[4]) {
  uint32_t pk[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float t0, t1;
    f2_unpack(f2_fma(f2_pack(x[2 * i], x[2 * i + 1]), sc2, nm2), t0, t1);
    const float p0 = ex2_approx(t0), p1 = ex2_approx(t1);
    acc[i & 3] = f2_add(acc[i & 3], f2_pack(p0, p1));
    pk[i] = pack_bf16x2(p0, p1);
  }
  tmem_st16(t_p, pk);
}

// Barrier of the softmax warps. Every one of them passes it equally often, whatever its waits
// returned: a warp that has given up skips the waits and the work, never the barriers.
__device__ __forceinline__ void softmax_barrier() {
  asm volatile("bar.sync 1, %0;" ::"n"(SOFTMAX_WARPS * 32) : "memory");
}

__device__ __forceinline__ uint32_t finite_only(uint32_t u) {
  if ((u & 0x7F80u) == 0x7F80u) u &= 0xFFFF0000u;
  if ((u & 0x7F800000u) == 0x7F800000u) u &= 0x0000FFFFu;
  return u;
}

// Thread `row` makes key row `row` of a V tile safe to multiply by zero: a row that nobody may
// read becomes zero; of a tree row in use only its infinities and NaN do, and the row is marked.
__device__ __forceinline__ void clean_v(Smem& s, uint32_t v, int row, bool clear, bool tree, int qb,
                                        int node) {
  const uint32_t addr = v + row * ROW_BYTES;
  if (clear) {
#pragma unroll
    for (int c = 0; c < 8; ++c) sts_u4(addr + c * 16, 0, 0, 0, 0);
  } else if (tree) {
    bool bad = false;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const uint4 u = lds_u4(addr + c * 16);
      if (has_nonfinite(u.x) || has_nonfinite(u.y) || has_nonfinite(u.z) || has_nonfinite(u.w)) {
        bad = true;
        sts_u4(addr + c * 16, finite_only(u.x), finite_only(u.y), finite_only(u.z),
               finite_only(u.w));
      }
    }
    if (bad) {
      atomicOr(&s.bad[qb][node >> 5], 1u << (node & 31));
      s.any_bad[qb] = 1;
    }
  }
  fence_proxy_async_smem();
}

// Adds to four columns of a row the visible tree V entries that are not finite (the finite entries of
// those V rows are in O already).
__device__ __forceinline__ void add_nonfinite(const Smem& s, const Params& p, int qb, const Unit& un,
                                           int row, int col, float4& n) {
  const uint32_t* see = s.mask[qb][row % p.t.N];
  for (int k = 0; k < MASK_WORDS; ++k) {
    for (uint32_t left = s.bad[qb][k] & see[k]; left != 0; left &= left - 1) {
      const __nv_bfloat16* src = p.t.tv + un.b * p.t.tv_sb + un.h * p.t.tv_sh +
                                 (k * 32 + __ffs(left) - 1) * p.t.tv_sn + col;
      const uint2 u = *reinterpret_cast<const uint2*>(src);
      if (!isfinite(bf16_lo(u.x))) n.x += bf16_lo(u.x);
      if (!isfinite(bf16_hi(u.x))) n.y += bf16_hi(u.x);
      if (!isfinite(bf16_lo(u.y))) n.z += bf16_lo(u.y);
      if (!isfinite(bf16_hi(u.y))) n.w += bf16_hi(u.y);
    }
  }
}

// Softmax and epilogue of warpgroup `group`: thread = TMEM lane = row `row` of copy `copy`.
template <int DUP>
__device__ __forceinline__ void softmax_role(Smem& s, const Params& p, uint32_t tmem, int warp,
                                             int lane) {
  constexpr int COLS = BM / DUP;   // keys of a tile that this copy works on
  constexpr int ROWS = BM / DUP;   // rows per copy
  constexpr int CHUNKS = COLS / 32;  // scores are handled 32 at a time: registers and code stay small
  const int group = warp >> 2, quarter = warp & 3;
  const int tid = quarter * 32 + lane;
  const int copy = tid / ROWS, row = tid % ROWS;
  const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
  const uint32_t t_s = tmem + lanes + S_COL + group * BM + copy * COLS;
  const uint32_t t_p = tmem + lanes + P_COL + group * (BM / 2) + copy * (COLS / 2);
  const uint32_t t_o = tmem + lanes + O_COL + group * HD;
  const float sl2 = p.t.scale_log2;
  const int R = p.t.G * p.t.N;
  uint32_t j = 0;  // tiles of this CTA so far
  bool ok = true;  // until a wait runs out
  Walk w;
  for (w.begin(p, s.start); w.left > 0; w.next(p)) {
    const int qb = w.seg & 1;
    ok = ok && warp_wait(&s.abort, &s.q_full[qb], (w.seg >> 1) & 1);
    const Unit un = s.unit[qb];
    const int row0 = un.row0, rows = ok ? un.rows : 0, L = un.len;
    const int node = ok ? (row0 + row) % p.t.N : 0;
    // Warps whose rows are all padding only keep the barriers going.
    const bool active = (quarter * 32) % ROWS < rows;
    float m_run = -INFINITY, l_run = 0.f;

    // Tile i of the unit, the CTA's j-th. Masked: a tile of the tree, or the cache's last one.
    auto step = [&](auto masked, int i) -> bool {
      const uint32_t use = j / GROUPS;
      const bool is_tree = i < p.tree_tiles;
      const int tile_key = (is_tree ? i : i - p.tree_tiles) * KEYS;
      if (!warp_wait(&s.abort, &s.s_full[group], use & 1)) return false;
      if constexpr (decltype(masked)::value) {
        const int st = static_cast<int>(j % V_STAGES);
        if (!warp_wait(&s.abort, &s.v_full[st], (j / V_STAGES) & 1)) return false;
        const int key = tile_key + tid;
        const bool clear = is_tree ? (key >= p.t.N || !node_used(s.mask[qb], key)) : key >= L;
        clean_v(s, smem_u32(s.v[st]), tid, clear, is_tree, qb, key);
      }
      tc_fence_after();
      float x[32];
      // 32 scores from TMEM, what is not visible at -inf. (Holding 64 spilled.)
      auto load = [&](int c) {
        uint32_t raw[32];
        tmem_ld32(t_s + c * 32, raw);
        tmem_wait_ld();
        reg_fence(raw);
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = __uint_as_float(raw[e]);
        if constexpr (decltype(masked)::value) {
          const int key0 = tile_key + copy * COLS + c * 32;
          uint32_t see;
          if (is_tree) {
            const int word = key0 >> 5;
            see = (row < rows && word < MASK_WORDS) ? s.mask[qb][node][word] : 0u;
          } else {
            const int n = L - key0;
            see = n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1u);
          }
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!((see >> e) & 1u)) x[e] = -INFINITY;
        }
      };
      float mx = -INFINITY;
      if (active) {
#pragma unroll
        for (int c = CHUNKS - 1; c >= 0; --c) {
          load(c);
          const float part = max32(x);
          mx = max3_nan(mx, part, part);
        }
      }
      auto scores_read = [&] {  // the last scores are in registers: the next ones may replace them
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.s_read[group]);
      };
      if (CHUNKS == 1 || !active) scores_read();
      // This warpgroup's previous product has read P and updated O.
      if (j >= GROUPS && !warp_wait(&s.abort, &s.pv_done[group], (use + 1) & 1)) return false;
      if (active) {
        const float m_new = max3_nan(m_run, mx * sl2, mx * sl2);
        bool rescale = false;
        float factor = 1.f;
        if (m_run == -INFINITY) {
          m_run = m_new;  // nothing seen so far: O and l are zero
        } else if (m_new > m_run + RESCALE_THRESHOLD || m_new != m_new) {
          rescale = true;
          factor = ex2_approx(m_run - m_new);
          m_run = m_new;
        }
        const float base = m_run == -INFINITY ? 0.f : m_run;
        const uint64_t sc2 = f2_pack(sl2, sl2), nm2 = f2_pack(-base, -base);
        uint64_t acc[4] = {0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
          if (c > 0) load(c);  // chunk 0 is still in x
          if (CHUNKS > 1 && c == CHUNKS - 1) scores_read();
          exp_store32(x, sc2, nm2, t_p + c * 16, acc);
        }
        acc[0] = f2_add(f2_add(acc[0], acc[1]), f2_add(acc[2], acc[3]));
        float lo, hi;
        f2_unpack(acc[0], lo, hi);
        const float sum = lo + hi;
        l_run = l_run * factor + sum;
        if (__any_sync(0xffffffffu, rescale)) {
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < HD; c += 32) {
            uint32_t o[32];
            tmem_ld32(t_o + c, o);
            tmem_wait_ld();
            reg_fence(o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
            tmem_st32(t_o + c, o);
          }
        }
        tmem_wait_st();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.p_ready[group]);
      return true;
    };
    // The warpgroups take the CTA's tiles alternately. Masked tiles: the tree's, and a last,
    // partial one of the cache.
    const int end = w.t0 + w.n;
    const int full_end = p.tree_tiles + L / KEYS;
    const uint32_t j_end = j + w.n;
    int last = -1;  // use of this warpgroup's last tile of the unit
    for (int i = w.t0; ok && i < end; ++i, ++j) {
      if ((j & (GROUPS - 1)) != static_cast<uint32_t>(group)) continue;
      last = static_cast<int>(j / GROUPS);
      if (i < p.tree_tiles || i >= full_end) ok = step(std::true_type{}, i);
      else ok = step(std::false_type{}, i);
    }
    j = j_end;

    // Epilogue: merge the GROUPS * DUP parts of every row, a block of columns at a time (unrolled
    // over the whole row this code ran once per unit out of a cold instruction cache and took
    // 5000 to 10000 cycles). SHARE threads write a row, WIDTH columns of the block each.
    constexpr int PARTS = GROUPS * DUP;
    constexpr int SHARE = SOFTMAX_WARPS * 32 / ROWS;   // threads that write one row
    constexpr int WIDTH = MERGE_COLS / SHARE;          // columns each of them has of a block
    const int part = group * DUP + copy;
    const int slot = part * ROWS + row;
    *reinterpret_cast<float2*>(s.ml[slot]) = make_float2(m_run, l_run);
    softmax_barrier();
    // A part that saw nothing has no O: its TMEM columns may hold another unit's.
    float M = -INFINITY;
#pragma unroll
    for (int k = 0; k < PARTS; ++k) M = fmaxf(M, s.ml[k * ROWS + row][0]);
    const float weight = last >= 0 ? merge_weight(m_run, M) : 0.f;
    const bool has_tree = w.t0 < p.tree_tiles;
    const bool whole = w.t0 == 0 && w.n == w.tiles;
    const bool any_bad = has_tree && s.any_bad[qb] != 0;
    const int out_row = static_cast<int>(threadIdx.x) / SHARE;
    const int out_col = static_cast<int>(threadIdx.x) % SHARE * WIDTH;
    float scale = 0.f;
    uint8_t* dst = nullptr;
    if (out_row < rows) {
      float m = -INFINITY, den = 0.f;
#pragma unroll
      for (int q = 0; q < PARTS; ++q) m = fmaxf(m, s.ml[q * ROWS + out_row][0]);
#pragma unroll
      for (int q = 0; q < PARTS; ++q) {
        const float2 ml = *reinterpret_cast<const float2*>(s.ml[q * ROWS + out_row]);
        den = fmaf(merge_weight(ml.x, m), ml.y, den);
      }
      const bool used = has_tree && node_used(s.mask[qb], (row0 + out_row) % p.t.N);
      if (whole) {
        const int64_t out = (static_cast<int64_t>(un.b) * p.t.Hkv + un.h) * R + row0 + out_row;
        const bool some = used && den != 0.f;
        scale = some ? 1.f / den : 0.f;
        dst = reinterpret_cast<uint8_t*>(p.t.o + out * HD + out_col);
        if (out_col == 0 && p.t.lse != nullptr)
          p.t.lse[out] = some ? (m + log2f(den)) * LN2 : -INFINITY;
      } else {
        float* rec = p.records + ((static_cast<int64_t>(blockIdx.x) * 2 + (w.t0 == 0 ? 1 : 0)) * p.rows +
                                  out_row) * REC;
        dst = reinterpret_cast<uint8_t*>(rec + out_col);
        if (out_col == 0)
          *reinterpret_cast<float4*>(rec + HD) = make_float4(m, den, used ? 1.f : 0.f, 0.f);
      }
    }
    if (last >= 0) ok = ok && warp_wait(&s.abort, &s.pv_done[group], last & 1);
    tc_fence_after();
    const uint32_t mine = smem_u32(s.merge[slot]);
    const uint32_t sums = smem_u32(s.merge[out_row]) + out_col * 4;
#pragma unroll 1
    for (int c0 = 0; c0 < HD; c0 += MERGE_COLS) {
      uint32_t o[MERGE_COLS];
      tmem_ld32(t_o + c0, o);
      tmem_wait_ld();
      reg_fence(o);
#pragma unroll
      for (int e = 0; e < MERGE_COLS; e += 4) {
        uint32_t y[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          y[k] = weight == 0.f ? 0u : __float_as_uint(__uint_as_float(o[e + k]) * weight);
        sts_u4(mine + e * 4, y[0], y[1], y[2], y[3]);
      }
      softmax_barrier();
      if (dst != nullptr) {
#pragma unroll
        for (int e = 0; e < WIDTH; e += 4) {
          float4 n = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int q = 0; q < PARTS; ++q) {
            const float4 x = lds_f4(sums + q * ROWS * MERGE_BYTES + e * 4);
            n.x += x.x;
            n.y += x.y;
            n.z += x.z;
            n.w += x.w;
          }
          if (any_bad) add_nonfinite(s, p, qb, un, row0 + out_row, c0 + out_col + e, n);
          if (whole)
            *reinterpret_cast<uint2*>(dst + (c0 + e) * 2) =
                scale != 0.f ? make_uint2(pack_bf16x2(n.x * scale, n.y * scale),
                                          pack_bf16x2(n.z * scale, n.w * scale))
                             : make_uint2(0, 0);
          else
            *reinterpret_cast<float4*>(dst + (c0 + e) * 4) = n;
        }
      }
      softmax_barrier();
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&s.q_free[qb]);
  }
}

// TMA producer (one thread).
__device__ __forceinline__ void load_role(Smem& s, const Params& p, const CUtensorMap& tm_k,
                                          const CUtensorMap& tm_v, const CUtensorMap& tm_tk,
                                          const CUtensorMap& tm_tv) {
  int ik = 0, iv = 0;
  bool ok = true;
  Walk w;
  for (w.begin(p, s.start); ok && w.left > 0; w.next(p)) {
    const int h = w.unit / p.t.row_tiles;
    for (int i = w.t0; i < w.t0 + w.n; ++i) {
      const bool is_tree = i < p.tree_tiles;
      const int key0 = (is_tree ? i : i - p.tree_tiles) * KEYS;
      const int ks = ik % K_STAGES, vs = iv % V_STAGES;
      if (ik >= K_STAGES &&
          !wait_or_abort(&s.abort, &s.k_empty[ks], ((ik / K_STAGES) + 1) & 1)) {
        ok = false;
        break;
      }
      mbar_arrive_expect_tx(&s.k_full[ks], TILE_BYTES);
      tma_load_4d(s.k[ks], is_tree ? &tm_tk : &tm_k, &s.k_full[ks], 0, key0, h, w.b);
      ++ik;
      if (iv >= V_STAGES &&
          !wait_or_abort(&s.abort, &s.v_empty[vs], ((iv / V_STAGES) + 1) & 1)) {
        ok = false;
        break;
      }
      mbar_arrive_expect_tx(&s.v_full[vs], TILE_BYTES);
      tma_load_4d(s.v[vs], is_tree ? &tm_tv : &tm_v, &s.v_full[vs], 0, key0, h, w.b);
      ++iv;
    }
  }
  if (s.abort) {
    // Never leave while a TMA write into this CTA's shared memory is pending.
    for (int c = max(0, ik - K_STAGES); c < ik; ++c)
      mbar_wait(&s.k_full[c % K_STAGES], (c / K_STAGES) & 1);
    for (int c = max(0, iv - V_STAGES); c < iv; ++c)
      mbar_wait(&s.v_full[c % V_STAGES], (c / V_STAGES) & 1);
  }
}

// Issues the scores S = Q K^T of every tile (one thread). Matrix descriptors differ in their start
// address only, so the loops add to one.
__device__ __forceinline__ void s_role(Smem& s, const Params& p, uint32_t tmem) {
  const uint32_t idesc = make_idesc_bf16(BM, KEYS, false);
  const uint64_t q0 = make_sdesc_sw128(smem_u32(s.q[0]), 16, 1024);
  const uint64_t k0 = make_sdesc_sw128(smem_u32(s.k[0]), 16, 1024);
  uint32_t buf = 0, st = 0, k_par = 0, read_par = 1;
  int used = 0;  // tiles issued so far, saturating
  bool ok = true;
  Walk w;
  for (w.begin(p, s.start); ok && w.left > 0; w.next(p)) {
    const int qb = w.seg & 1;
    if (!wait_or_abort(&s.abort, &s.q_full[qb], (w.seg >> 1) & 1)) break;
    const uint64_t a = q0 + qb * (TILE_BYTES >> 4);
    for (int i = 0; i < w.n; ++i) {
      if (!wait_or_abort(&s.abort, &s.k_full[st], k_par) ||
          (used == GROUPS && !wait_or_abort(&s.abort, &s.s_read[buf], read_par))) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint64_t b = k0 + st * (TILE_BYTES >> 4);
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk)
        umma_ss(tmem + S_COL + buf * BM, a + kk * 2, b + kk * 2, idesc, kk > 0 ? 1u : 0u);
      umma_commit(&s.s_full[buf]);
      umma_commit(&s.k_empty[st]);
      if (used < GROUPS) ++used;
      if (++st == K_STAGES) {
        st = 0;
        k_par ^= 1u;
      }
      if (++buf == GROUPS) {
        buf = 0;
        read_par ^= 1u;
      }
    }
    umma_commit(&s.q_free[qb]);
  }
  // All products issued by this thread have completed once its drain barrier flips.
  umma_commit(&s.drain[0]);
  mbar_wait(&s.drain[0], 0);
}

// Issues O += P V of every tile (one thread): 8 steps of 16 keys, P from TMEM (8 columns a step).
__device__ __forceinline__ void pv_role(Smem& s, const Params& p, uint32_t tmem) {
  const uint32_t idesc = make_idesc_bf16(BM, HD, true);
  const uint64_t v0 = make_sdesc_sw128(smem_u32(s.v[0]), 8192, 1024);
  uint32_t buf = 0, st = 0, v_par = 0, p_par = 0;
  bool ok = true;
  Walk w;
  for (w.begin(p, s.start); ok && w.left > 0; w.next(p)) {
    // O of the previous unit has been read before P of this one's first tiles is there.
    for (int i = 0; i < w.n; ++i) {
      if (!wait_or_abort(&s.abort, &s.v_full[st], v_par) ||
          !wait_or_abort(&s.abort, &s.p_ready[buf], p_par)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint64_t b = v0 + st * (TILE_BYTES >> 4);
      const uint32_t d = tmem + O_COL + buf * HD, a = tmem + P_COL + buf * (BM / 2);
#pragma unroll
      for (int kk = 0; kk < KEYS / 16; ++kk)
        umma_ts(d, a + kk * 8, b + kk * 128, idesc, (i >= GROUPS || kk > 0) ? 1u : 0u);
      umma_commit(&s.pv_done[buf]);
      umma_commit(&s.v_empty[st]);
      if (++st == V_STAGES) {
        st = 0;
        v_par ^= 1u;
      }
      if (++buf == GROUPS) {
        buf = 0;
        p_par ^= 1u;
      }
    }
  }
  umma_commit(&s.drain[1]);
  mbar_wait(&s.drain[1], 0);
}

// Q (DUP copies, zero rows in between), the unit's numbers and, where its part has tiles of the tree,
// the ancestor masks into buffer qb, by `threads` threads. `sync` as in build_masks; `built` is the
// batch row whose masks the buffer holds.
template <int DUP, typename Sync>
__device__ __forceinline__ void load_unit(Smem& s, const Params& p, const Walk& w, int qb, int tid,
                                          int threads, int& built, Sync sync) {
  constexpr int ROWS = BM / DUP;
  const int h = w.unit / p.t.row_tiles;
  const int row0 = (w.unit - h * p.t.row_tiles) * p.rows;
  const int rows = min(p.rows, p.t.G * p.t.N - row0);
  const uint32_t base = smem_u32(s.q[qb]);
  // Asynchronous 16-byte copies, all in flight at once (size 0 fills with zeros): 8 threads a row.
  const int c = tid & 7;
  const __nv_bfloat16* head =
      p.t.q + w.b * p.t.q_sb + static_cast<int64_t>(h) * p.t.G * p.t.q_sh + c * 8;
  int g = (row0 + (tid >> 3)) / p.t.N, n = row0 + (tid >> 3) - g * p.t.N;
  for (int r = tid >> 3; r < ROWS; r += threads >> 3) {
    const bool in = r < rows;
    const __nv_bfloat16* src = in ? head + g * p.t.q_sh + n * p.t.q_sn : head;
#pragma unroll
    for (int k = 0; k < DUP; ++k) {
      const int at = k * ROWS + r;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                       base + at * ROW_BYTES + ((c ^ (at & 7)) << 4)),
                   "l"(src), "r"(in ? 16 : 0)
                   : "memory");
    }
    for (n += threads >> 3; n >= p.t.N; n -= p.t.N) ++g;
  }
  if (tid == 0) s.unit[qb] = Unit{w.b, h, row0, rows, valid_len(p.t.lens, p.t.C, w.b)};
  if (w.t0 < p.tree_tiles) {
    const int b = p.t.parents_sb == 0 ? 0 : w.b;
    if (built != b) {
      build_masks(p.t.parents + b * p.t.parents_sb, p.t.N, s.jump, s.mask[qb], tid, threads, sync);
      built = b;
    }
    if (tid < MASK_WORDS) s.bad[qb][tid] = 0;
    if (tid == 0) s.any_bad[qb] = 0;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  fence_proxy_async_smem();
}

// The units from the second on, up to two ahead (one warp; the softmax warps load the first one
// together, since nothing can begin before it).
template <int DUP>
__device__ __forceinline__ void q_role(Smem& s, const Params& p, int lane) {
  int built[2] = {-1, -1};
  Walk w;
  w.begin(p, s.start);
  if (w.left > 0) w.next(p);
  for (; w.left > 0; w.next(p)) {
    const int qb = w.seg & 1;
    // Also keeps this warp's use of s.jump behind the first unit's.
    if (w.seg == 1 && !warp_wait(&s.abort, &s.q_full[0], 0)) break;
    if (w.seg >= 2 && !warp_wait(&s.abort, &s.q_free[qb], ((w.seg >> 1) + 1) & 1)) break;
    load_unit<DUP>(s, p, w, qb, lane, 32, built[qb],
                   [](bool any) {
                     __syncwarp();  // a vote alone orders no memory
                     return __any_sync(0xffffffffu, any) != 0;
                   });
    __syncwarp();
    if (lane == 0) mbar_arrive(&s.q_full[qb]);
  }
}

template <int DUP>
__global__ void __launch_bounds__(THREADS, 1)
tree_persistent_kernel(const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v,
                       const __grid_constant__ CUtensorMap tm_tk,
                       const __grid_constant__ CUtensorMap tm_tv, const Params p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem& s = *reinterpret_cast<Smem*>(smem_raw);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  // The next kernel (the merge) may be scheduled from here on; it waits for this grid to complete.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (warp == 0) {
    wait_for_previous_kernel();
    const Start st = find_start(p, blockIdx.x, gridDim.x, lane);
    if (lane == 0) {
      s.start = st;
      p.starts[blockIdx.x] = st;
    }
  } else if (warp == S_WARP) {
    tmem_alloc(&s.tmem_base, TMEM_COLS);
    tmem_relinquish();
  } else if (threadIdx.x == LOAD_WARP * 32) {
    for (int i = 0; i < K_STAGES; ++i) {
      mbar_init(&s.k_full[i], 1);
      mbar_init(&s.k_empty[i], 1);
    }
    for (int i = 0; i < V_STAGES; ++i) {
      mbar_init(&s.v_full[i], 1);
      mbar_init(&s.v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.q_full[i], 1);
      mbar_init(&s.q_free[i], 1 + SOFTMAX_WARPS);
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.s_read[i], 4);
      mbar_init(&s.p_ready[i], 4);
      mbar_init(&s.pv_done[i], 1);
      mbar_init(&s.drain[i], 1);
    }
    s.abort = 0;
    fence_barrier_init();
  }
  if (warp != 0) wait_for_previous_kernel();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem_base;
  if (warp < SOFTMAX_WARPS) {
    // P starts as zero: the entries of other copies' keys stay so.
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    uint32_t z[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) z[i] = 0;
#pragma unroll
    for (int c = 0; c < 2; ++c)
      tmem_st32(tmem + lanes + P_COL + (warp >> 2) * (BM / 2) + c * 32, z);
    tmem_wait_st();
    tc_fence_before();
    Walk first;
    first.begin(p, s.start);
    if (first.left > 0) {
      int built = -1;
      load_unit<DUP>(s, p, first, 0, threadIdx.x, SOFTMAX_WARPS * 32, built,
                     [](bool any) { return barrier_or<SOFTMAX_WARPS * 32>(any); });
      softmax_barrier();
      if (threadIdx.x == 0) mbar_arrive(&s.q_full[0]);
    }
    softmax_role<DUP>(s, p, tmem, warp, lane);
  } else {
    if (warp == LOAD_WARP) {
      if (lane == 0) load_role(s, p, tm_k, tm_v, tm_tk, tm_tv);
    } else if (warp == S_WARP) {
      if (lane == 0) s_role(s, p, tmem);
    } else if (warp == PV_WARP) {
      if (lane == 0) pv_role(s, p, tmem);
    } else {
      q_role<DUP>(s, p, lane);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == S_WARP) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

// Merge of the units that lie in more than one CTA. Block (c, g) looks at the boundary between
// CTAs c and c + 1: if it is the first one inside a unit, the block merges that unit's records
// for rows [8 g, 8 g + 8), 8 threads a row for the columns and two shares of the records, whose
// loads are all in flight together (a thread per row and column walking 13 records took 8 us). It
// takes 6 us: the end of the grid before it, the starts, the records, the rows, one after another. (A
// block per shared unit instead, found from all starts, costs 1.5 us more; half the registers and
// twice the blocks per SM change less than 1 us either way.)
__global__ void __launch_bounds__(COMBINE_THREADS) tree_combine_kernel(const Params p, int grid) {
  wait_for_previous_kernel();
  const int c = static_cast<int>(blockIdx.x);
  const int lane = threadIdx.x & 31;
  // Lane k looks at CTA c + k: the pieces are the CTAs after c that began inside the same unit.
  Start own{};
  if (c + lane < grid) own = p.starts[c + lane];
  const int unit_b = __shfl_sync(0xffffffffu, own.b, 1);
  const int unit_u = __shfl_sync(0xffffffffu, own.unit, 1);
  unsigned inside = __ballot_sync(0xffffffffu, own.count > 0 && own.tile > 0 && own.b == unit_b &&
                                                   own.unit == unit_u);
  // CTA c itself inside the same unit: an earlier block has it (c = 0 never is).
  if (!(inside & 2u) || (inside & 1u)) return;
  int pieces = __ffs(~(inside >> 1));  // 1 + the run of CTAs from c + 1 on (32 lanes seen: 31)
  if (pieces == 32) {
    while (c + pieces < grid) {
      const Start s = p.starts[c + pieces];
      if (s.count == 0 || s.tile == 0 || s.b != unit_b || s.unit != unit_u) break;
      ++pieces;
    }
  }
  const int R = p.t.G * p.t.N;
  const int row0 = (unit_u % p.t.row_tiles) * p.rows;
  const int rows = min(p.rows, R - row0);
  const int r_in = static_cast<int>(threadIdx.x >> 3) % COMBINE_ROWS;
  const int share = static_cast<int>(threadIdx.x >> 3) / COMBINE_ROWS;
  const int r = static_cast<int>(blockIdx.y) * COMBINE_ROWS + r_in;
  const int c8 = threadIdx.x & 7;
  const bool in_unit = r < rows;
  const float* first = p.records + (static_cast<int64_t>(c) * 2 * p.rows + (in_unit ? r : 0)) * REC;
  const int64_t step = static_cast<int64_t>(2) * p.rows * REC;
  float M = -INFINITY, den = 0.f, n[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  float used = 0.f;
  constexpr int BATCH = 8;
  for (int k0 = share; k0 < pieces; k0 += BATCH * COMBINE_SHARES) {
    float4 ml[BATCH], x[BATCH], y[BATCH];
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const int at = k0 + k * COMBINE_SHARES;
      const bool in = at < pieces;
      // The first piece is in its CTA's second record, the others in their first.
      const float4* src = reinterpret_cast<const float4*>(first + (in ? at : 0) * step +
                                                          (in && at > 0 ? 0 : p.rows * REC));
      ml[k] = in ? src[HD / 4] : make_float4(-INFINITY, 0.f, 0.f, 0.f);
      x[k] = in ? src[c8 * 2] : make_float4(0.f, 0.f, 0.f, 0.f);
      y[k] = in ? src[c8 * 2 + 1] : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    if (k0 == 0) used = ml[0].z;
    float m_new = M;
#pragma unroll
    for (int k = 0; k < BATCH; ++k) m_new = fmaxf(m_new, ml[k].x);
    const float f = merge_weight(M, m_new);
    M = m_new;
    den *= f;
#pragma unroll
    for (int e = 0; e < 8; ++e) n[e] *= f;
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const float wt = merge_weight(ml[k].x, M);
      den = fmaf(wt, ml[k].y, den);
      n[0] = fmaf(wt, x[k].x, n[0]); n[1] = fmaf(wt, x[k].y, n[1]);
      n[2] = fmaf(wt, x[k].z, n[2]); n[3] = fmaf(wt, x[k].w, n[3]);
      n[4] = fmaf(wt, y[k].x, n[4]); n[5] = fmaf(wt, y[k].y, n[5]);
      n[6] = fmaf(wt, y[k].z, n[6]); n[7] = fmaf(wt, y[k].w, n[7]);
    }
  }
  // The second share's result to the first.
  __shared__ float part[COMBINE_SHARES - 1][COMBINE_ROWS * 8][10];
  if (share > 0) {
    float* dst = part[share - 1][r_in * 8 + c8];
#pragma unroll
    for (int e = 0; e < 8; ++e) dst[e] = n[e];
    dst[8] = M;
    dst[9] = den;
  }
  __syncthreads();
  if (share > 0 || !in_unit) return;
#pragma unroll
  for (int k = 0; k < COMBINE_SHARES - 1; ++k) {
    const float* src = part[k][r_in * 8 + c8];
    const float m_new = fmaxf(M, src[8]);
    const float a = merge_weight(M, m_new), w = merge_weight(src[8], m_new);
    M = m_new;
    den = den * a + src[9] * w;
#pragma unroll
    for (int e = 0; e < 8; ++e) n[e] = n[e] * a + src[e] * w;
  }
  const int bh = unit_b * p.t.Hkv + unit_u / p.t.row_tiles;
  write_out(p.t, static_cast<int64_t>(bh) * R + row0 + r, c8, n, M, den, used != 0.f);
}

}  // namespace persist
}  // namespace tree
}  // namespace tt
