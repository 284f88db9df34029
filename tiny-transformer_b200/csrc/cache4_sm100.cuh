// KV cache held in 4 bits: its format, the kernel that norms, turns, quantises and writes the rows of a fused
// QKV projection, and the kernel that reads rows back as bf16, sm_100a.
//
// Format. A cache is [B, Hkv, blocks, 576] bytes; a block holds 16 rows (tokens) of 64 features: 512 bytes of codes
// (row r at 32 r, feature 2i in the low half of byte i), then 64 bytes of scales (row r at 512 + 4 r, one for 16
// features). A code is e2m1 (sign, 0 0.5 1 1.5 2 3 4 6). A scale is the upper byte of a half without its sign: 5
// bits of exponent and 3 of mantissa, 2^-17 to 10240 here. A value is code x scale, exact in half precision
// and in bf16 (2 + 4 significant bits). The five exponent bits make a scale for the whole tensor unnecessary:
// scales have four significant bits from 2^-14 on, for groups whose largest value is at least 3.7e-4 (with 4 exponent bits:
// 0.09), lose them one by one below that, and groups below 2.3e-5 become zero. A scale becomes a half by a shift.
//
// Quantising 16 values x: scale = max|x| / 6 rounded to nearest even (to 10240 at most), code = x / scale rounded to
// nearest, ties to the even code, saturating at 6. Values are bf16, so borders are exact numbers: a tie x =
// border x scale (3 x 4 bits) is a bf16 number, every other bf16 number is at least 2^-8 of itself away, and
// x * (1 / scale) is off by 2^-21 of itself at most; rounding it to multiples of 2^-13 restores ties and crosses none.
// In the same way max|x| times 1/6 is off by 2^-23, a tie of the scale has 5 significant bits, and rounding to 20 bits
// first restores it. A group with a NaN gets the scale NaN; infinities saturate.
//
// Append: key rows are quantised from the bf16 values of the rotation, rounded from 64 bits by way of FP32 (as double goes to
// bf16 in two conversions): an error of the last bit next to a border would be a whole step of a code. FP32 decides wherever a value is farther from a bf16 border
// than its error bound. Of the others (one in 2^10) both neighbours are quantised, and where that gives different
// codes the row is computed again in FP64.
//
// Memory: append 128 bytes a head in, 128 or 36 out; read 36 in, 128 out. Measured (B200, 4 x 4096 tokens of 12 + 12 + 12
// heads): append 31 us (115 MB, 3.7 TB/s; its integer and conversion instructions bound it, 200 a head of four
// rows; 43.7 us with keys, values and queries mixed in a CTA and every doubtful row in FP64), read back 14 us
// (4.6 TB/s, conversions again). A decode step of 64 sequences: append and read back of its rows 4.3 us.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "norm_rope_sm100.cuh"
#include "sm100_ptx.cuh"

namespace tt {
namespace cache4 {

constexpr int HD = 64;
constexpr int BLOCK_ROWS = 16;
constexpr int CODE_BYTES = BLOCK_ROWS * HD / 2;         // 512
constexpr int GROUPS = 4;                               // scales of a row
constexpr int BLOCK_BYTES = CODE_BYTES + BLOCK_ROWS * GROUPS;
constexpr int MAX_QUERIES = 16;
constexpr uint32_t MAX_SCALE_BYTE = 0xe2;               // 10240

struct View {   // a cache: byte strides of batch, head and block
  uint8_t* p;
  int64_t sb, sh, sn;
};

// Eight codes of a word as four half pairs: pair i holds features 2i (low) and 2i + 1.
__device__ __forceinline__ void decode8(uint32_t w, uint32_t (&r)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
      : "r"(w));
}

__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// A scale byte as a pair of equal halves.
__device__ __forceinline__ uint32_t scale_pair(uint32_t byte) { return byte * 0x00800080u; }

// ------------------------------------------------------------------------------- quantising

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// Eight bf16 values (this lane's half of a group of 16; the other half is in lane ^ 1) to a word of codes.
// Returns the group's scale byte.
__device__ __forceinline__ uint32_t quantise8(const uint4& v, uint32_t& codes) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
  // Largest |x| as bits: a NaN is above infinity.
  uint32_t two = max_u16x2(max_u16x2(u[0] & 0x7fff7fffu, u[1] & 0x7fff7fffu),
                           max_u16x2(u[2] & 0x7fff7fffu, u[3] & 0x7fff7fffu));
  two = max_u16x2(two, __shfl_xor_sync(0xffffffffu, two, 1));
  const uint32_t top = max(two & 0xffffu, two >> 16);
  const uint32_t sixth = __float_as_uint(__uint_as_float(top << 16) * (1.0f / 6.0f));
  // Times 2^-112 a float's exponent and mantissa are those of the scale byte, subnormals included.
  const uint32_t bits = __float_as_uint(__uint_as_float((sixth + 8u) & ~15u) * 1.92592994438723586e-34f);
  uint32_t byte = min((bits + 0x7ffffu + ((bits >> 20) & 1u)) >> 20, MAX_SCALE_BYTE);
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(__uint_as_float(byte << 20) * 5.192296858534828e33f));
  if (byte == 0) inv = 0.0f;
  if (top > 0x7f80u) byte = 0xffu;
  float y[8];
  const uint64_t inv2 = f2_pack(inv, inv);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t x = f2_pack(bf16_lo(u[i]), bf16_hi(u[i]));
    f2_unpack(f2_add(f2_fma(x, inv2, f2_pack(1536.0f, 1536.0f)), f2_pack(-1536.0f, -1536.0f)), y[2 * i],
              y[2 * i + 1]);
  }
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(codes)
      : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
  return byte;
}

// Where a lane's part of a row stands in each head of a cache: 4 bytes of codes, and the row's scales.
struct RowPlace {
  uint8_t* codes;
  uint8_t* scales;

  __device__ __forceinline__ void set(const View& c, int b, int64_t pos, int lane8) {
    uint8_t* block = c.p + b * c.sb + (pos / BLOCK_ROWS) * c.sn;
    const int r = static_cast<int>(pos % BLOCK_ROWS);
    codes = block + r * (HD / 2) + lane8 * 4;
    scales = block + CODE_BYTES + r * GROUPS;
  }
};

// Stores a row's codes and scales (each lane its word and its group's byte).
__device__ __forceinline__ void store_row(const RowPlace& at, int64_t head, int lane8, bool ok, uint32_t codes,
                                          uint32_t byte) {
  uint32_t scales = (lane8 & 1) ? 0u : byte << (4 * lane8);
  scales |= __shfl_xor_sync(0xffffffffu, scales, 2);
  scales |= __shfl_xor_sync(0xffffffffu, scales, 4);
  if (!ok) return;
  *reinterpret_cast<uint32_t*>(at.codes + head) = codes;
  if (lane8 == 0) *reinterpret_cast<uint32_t*>(at.scales + head) = scales;
}

// ------------------------------------------------------------------------------- append

struct AppendParams {
  norm_rope::Common c;
  __nv_bfloat16* q_out;   // [B, Hq, T, 64]
  View cache[2];          // keys, values
  int64_t capacity;       // rows
};

// The bf16 values of a key row from FP32, `up` those from above; they differ where FP32 cannot tell how a value is
// rounded. False for a row whose mean square leaves FP32's safe range. `most` is the largest coefficient of each
// pair, times 2^-20.
template <bool NORM>
__device__ __forceinline__ bool key_row(const uint4& v, const norm_rope::Coefficients& k, const uint64_t (&most)[2],
                                        float eps, uint4& out, uint4& up) {
  norm_rope::Pairs x;
  x.unpack(v);
  const float r = NORM ? norm_rope::inverse_rms(x, eps) : 1.0f;
  if (NORM) x.scale(r);
  const norm_rope::Pairs y = k.turn(x);
  norm_rope::Pairs lo, hi;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    // An element's terms are below (|x_2i| + |x_2i+1|) most; in units of 2^-20 of that it is off by: rsqrtf .25,
    // the sum of squares .25 (8 roundings), eps .03, five more roundings .0625 each, and the one here.
    float e0, e1, o0, o1;
    f2_unpack(x.e[i], e0, e1);
    f2_unpack(x.o[i], o0, o1);
    const uint64_t size = f2_pack(fabsf(e0) + fabsf(o0), fabsf(e1) + fabsf(o1));
    const uint64_t off = f2_mul(size, most[i]), minus = f2_pack(-1.0f, -1.0f);
    lo.e[i] = f2_fma(off, minus, y.e[i]);
    lo.o[i] = f2_fma(off, minus, y.o[i]);
    hi.e[i] = f2_add(off, y.e[i]);
    hi.o[i] = f2_add(off, y.o[i]);
  }
  out = lo.pack();
  up = hi.pack();
  return r > 1e-15f && r < 1e15f;
}

__device__ __forceinline__ uint32_t min_u16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("min.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// Two candidates for each value to the smaller and the larger magnitudes (zero below candidates of different signs). The
// true row lies between these in every place, and scales and codes grow with magnitudes: where both have the same, it
// has them too (but for the sign of a zero).
__device__ __forceinline__ void order(uint4& a, uint4& b) {
  uint32_t* x[4] = {&a.x, &a.y, &a.z, &a.w};
  uint32_t* y[4] = {&b.x, &b.y, &b.z, &b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t sign = *x[i] & 0x80008000u, p = *x[i] & 0x7fff7fffu, q = *y[i] & 0x7fff7fffu;
    const uint32_t crossed = (((*x[i] ^ *y[i]) >> 15) & 0x00010001u) * 0xffffu;
    *x[i] = (min_u16x2(p, q) & ~crossed) | sign;
    *y[i] = max_u16x2(p, q) | sign;
  }
}

// The same from FP64, rounded to FP32 and then to bf16 (two roundings: within 2^-25 of a bf16 tie the second is a tie).
template <bool NORM>
__device__ __forceinline__ uint4 key_row_exact(const norm_rope::Common& p, const uint4& v, int64_t pos, int lane8) {
  constexpr int E = norm_rope::E;
  float x[E], w[E];
  norm_rope::unpack8(v, x);
  norm_rope::Turn u;
  norm_rope::load_turn(p, pos, lane8, u);
#pragma unroll
  for (int i = 0; i < E; ++i) w[i] = 1.0f;
  double r = 1.0;
  if (NORM) {
    norm_rope::load_weight(p, 1, lane8, w);
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < E; ++i) ss += static_cast<double>(x[i]) * x[i];
#pragma unroll
    for (int m = 1; m < 8; m *= 2) ss += __shfl_xor_sync(0xffffffffu, ss, m);
    r = 1.0 / sqrt(ss / HD + p.eps);
  }
  uint32_t y[4];
#pragma unroll
  for (int i = 0; i < E / 2; ++i) {
    const double a = x[2 * i] * r * w[2 * i], b = x[2 * i + 1] * r * w[2 * i + 1];
    const double c = u.c[i], s = u.s[i];
    y[i] = pack_bf16x2(static_cast<float>(a * c - b * s), static_cast<float>(a * s + b * c));
  }
  return make_uint4(y[0], y[1], y[2], y[3]);
}

template <bool NORM>
__global__ void __launch_bounds__(norm_rope::THREADS, 7)
    append_kernel(const __grid_constant__ AppendParams ap) {
  namespace nr = norm_rope;
  const nr::Common& p = ap.c;
  const int lane = threadIdx.x & 31, lane8 = lane & 7;
  // Keys first: they take longest.
  int index = static_cast<int>(blockIdx.x) * nr::WARPS + (threadIdx.x >> 5), kind = 1;
  wait_for_previous_kernel();
  if (index >= p.total[1]) {
    index -= p.total[1];
    kind = 2;
    if (index >= p.total[2]) {
      index -= p.total[2];
      kind = 0;
    }
  }
  if (index >= p.total[kind]) return;  // whole warps
  nr::Item it;
  it.set(p, kind, index, lane);
  const __nv_bfloat16* src = p.qkv + it.b * p.x_sb + static_cast<int64_t>(it.row ? it.t : 0) * p.x_st +
                             it.head0(p) * p.x_sh + lane8 * nr::E;
  nr::HeadRows<nr::SMALL_BATCH> in;
  in.start(src, p.x_sh, it.heads);
  const int64_t pos = it.row ? nr::position_of(p, it.b, it.t) : 0;
  const bool ok = it.row && pos >= 0 && pos < p.table_len && pos < ap.capacity;
  if (it.row && !ok && lane8 == 0) atomicOr(&g_tt_status, TT_ERR_RANGE);
  const int64_t at = ok ? pos : 0;
  if (it.kind == 2) {
    RowPlace place;
    place.set(ap.cache[1], it.b, at, lane8);
    int64_t head = it.first * ap.cache[1].sh;
    do {
      in.prefetch();
#pragma unroll
      for (int j = 0; j < nr::SMALL_BATCH; ++j, head += ap.cache[1].sh)
        if (j < in.left) {
          uint32_t codes;
          const uint32_t byte = quantise8(in.now[j], codes);
          store_row(place, head, lane8, ok, codes, byte);
        }
    } while (in.advance());
    return;
  }
  nr::Turn u;
  nr::load_turn(p, at, lane8, u);
  nr::Coefficients k;
  k.set<NORM>(p, it.kind, u, lane8);
  const float eps = static_cast<float>(p.eps);
  if (it.kind == 0) {
    nr::turn_heads<NORM>(
        in, k, eps,
        ap.q_out + ((static_cast<int64_t>(it.b) * p.Hq + it.first) * p.T + it.t) * HD + lane8 * nr::E,
        static_cast<int64_t>(p.T) * HD, it.row, ok);
    return;
  }
  RowPlace place;
  place.set(ap.cache[0], it.b, at, lane8);
  uint64_t most[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float a[4], b[4];
    f2_unpack(k.ec[i], a[0], b[0]);
    f2_unpack(k.es[i], a[1], b[1]);
    f2_unpack(k.oc[i], a[2], b[2]);
    f2_unpack(k.os[i], a[3], b[3]);
    constexpr float UNIT = 9.5367431640625e-07f;   // 2^-20
    most[i] = f2_pack(UNIT * fmaxf(fmaxf(fabsf(a[0]), fabsf(a[1])), fmaxf(fabsf(a[2]), fabsf(a[3]))),
                      UNIT * fmaxf(fmaxf(fabsf(b[0]), fabsf(b[1])), fmaxf(fabsf(b[2]), fabsf(b[3]))));
  }
  unsigned unsure = 0;   // heads
  int64_t head = it.first * ap.cache[0].sh;
  int h = 0;
  do {
    in.prefetch();
#pragma unroll
    for (int j = 0; j < nr::SMALL_BATCH; ++j, ++h, head += ap.cache[0].sh) {
      if (j >= in.left) break;
      uint4 y, up;
      const bool safe = key_row<NORM>(in.now[j], k, most, eps, y, up);
      uint32_t codes, byte;
      const bool sure = safe && ((y.x ^ up.x) | (y.y ^ up.y) | (y.z ^ up.z) | (y.w ^ up.w)) == 0;
      if (__any_sync(0xffffffffu, !sure)) {
        order(y, up);
        uint32_t above;
        const uint32_t byte_above = quantise8(up, above);
        byte = quantise8(y, codes);
        if (__any_sync(0xffffffffu, !safe || codes != above || byte != byte_above)) unsure |= 1u << h;
      } else {
        byte = quantise8(y, codes);
      }
      store_row(place, head, lane8, ok, codes, byte);
    }
  } while (in.advance());
  while (unsure != 0) {
    h = __ffs(static_cast<int>(unsure)) - 1;
    unsure &= unsure - 1;
    const uint4 x = *reinterpret_cast<const uint4*>(src + h * p.x_sh);
    uint32_t codes;
    const uint32_t byte = quantise8(key_row_exact<NORM>(p, x, at, lane8), codes);
    store_row(place, (it.first + h) * ap.cache[0].sh, lane8, ok, codes, byte);
  }
}

// ------------------------------------------------------------------------------- read

struct ReadParams {
  View cache[2];
  __nv_bfloat16* out[2];          // [B, Hkv, rows, 64]
  int B, Hkv, rows;
  norm_rope::Divisor chunks, heads;   // divisions by the chunks of 16 rows of a head, by Hkv
  int64_t capacity;
  int64_t start;                  // first row where start_dev is NULL
  const int64_t* start_dev;       // first row of sequence b: start_dev[b * start_sb]
  int64_t start_sb;
};

constexpr int READ_WARPS = 4;
// Rows of a warp: four steps of four, all loads in flight together (64 rows took 11.3 us against 7.4 for the append and
// read back of 3 x 1058 rows of 4 heads, and 46 against 44 for 4 x 4096 of 12).
constexpr int READ_ROWS = 16;

// Eight lanes a row: 4 bytes of codes and the group's scale each, 16 bytes out.
__global__ void __launch_bounds__(READ_WARPS * 32) read_kernel(const __grid_constant__ ReadParams p) {
  constexpr int STEPS = READ_ROWS / 4;
  const int lane = threadIdx.x & 31, lane8 = lane & 7;
  wait_for_previous_kernel();
  // Item: (K or V, sequence, head, 16 rows).
  const unsigned index = blockIdx.x * READ_WARPS + (threadIdx.x >> 5);
  const unsigned row_of = p.chunks.of(static_cast<int>(index)), heads = static_cast<unsigned>(p.B) * p.Hkv;
  if (row_of >= 2 * heads) return;   // whole warps
  const int kv = row_of >= heads ? 1 : 0;
  const int bh = static_cast<int>(row_of - kv * heads);
  const int b = p.heads.of(bh), h = bh - b * p.Hkv;
  const int first = static_cast<int>(index - row_of * p.chunks.d) * READ_ROWS + (lane >> 3);
  const View& c = p.cache[kv];
  const int64_t start = p.start_dev != nullptr ? p.start_dev[b * p.start_sb] : p.start;
  // Rows and the capacity are below 2^31; a start far outside must not wrap.
  const int64_t far = int64_t(1) << 40;
  const int at = static_cast<int>(min(max(min(max(start, -far), far) + first, int64_t(-64)), p.capacity));
  // Rows are at most 12 behind `at`, so in its block or the next one.
  const uint8_t* block = c.p + b * c.sb + h * c.sh + static_cast<int64_t>(max(at, 0) / BLOCK_ROWS) * c.sn;
  const int in = max(at, 0) % BLOCK_ROWS - max(at, 0);
  uint32_t codes[STEPS], byte[STEPS];
  bool outside = false;
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    codes[s] = byte[s] = 0;
    if (first + 4 * s >= p.rows) continue;
    const int pos = at + 4 * s;
    if (pos < 0 || pos >= p.capacity) {   // reads as zero
      outside = true;
      continue;
    }
    const int r = pos + in;   // row from the start of `block`
    const uint8_t* from = block + (r >= BLOCK_ROWS ? c.sn : 0);
    codes[s] = *reinterpret_cast<const uint32_t*>(from + r % BLOCK_ROWS * (HD / 2) + lane8 * 4);
    byte[s] = from[CODE_BYTES + r % BLOCK_ROWS * GROUPS + (lane8 >> 1)];
  }
  if (outside && lane8 == 0) atomicOr(&g_tt_status, TT_ERR_RANGE);
  __nv_bfloat16* out = p.out[kv] + (static_cast<int64_t>(bh) * p.rows + first) * HD + lane8 * 8;
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    if (first + 4 * s >= p.rows) break;
    uint32_t pairs[4], y[4];
    decode8(codes[s], pairs);
    const uint32_t scale = scale_pair(byte[s]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t two = mul_half2(pairs[i], scale);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&two));
      y[i] = pack_bf16x2(f.x, f.y);
    }
    *reinterpret_cast<uint4*>(out + s * 4 * HD) = make_uint4(y[0], y[1], y[2], y[3]);
  }
}

}  // namespace cache4
}  // namespace tt
