// KV cache held in 4 bits: its format, the kernel that norms, turns, quantises and writes the rows of a fused
// QKV projection, and the kernel that reads rows back as bf16, sm_100a.
//
// Format. A cache is [B, Hkv, blocks, 576] bytes; a block holds 16 rows (tokens) of 64 features: 512 bytes of codes
// (row r at 32 r, feature 2i in the low half of byte i), then 64 bytes of scales (row r at 512 + 4 r, one for 16
// features). A code is e2m1 (sign, 0 0.5 1 1.5 2 3 4 6). A scale is the upper byte of a half without its sign: 5
// bits of exponent and 3 of mantissa, 2^-17 to 10240 here. A value is code x scale, exact in half precision
// and in bf16 (2 + 4 significant bits). The five exponent bits make a scale for the whole tensor unnecessary
// (with 4, a group whose largest value is below 0.09 would lose bits), and a scale becomes a half by a shift.
//
// Quantising 16 values x: scale = max|x| / 6 rounded to nearest even (to 10240 at most), code = x / scale rounded to
// nearest, ties to the even code, saturating at 6. Values are bf16, so borders are exact: a tie x = border x scale
// (3 x 4 bits) is a bf16 number, every other bf16 number is at least 2^-8 of itself away, and the product
// x * (1 / scale) is off by 2^-22 of itself at most. Rounding it to multiples of 2^-13 restores ties and
// crosses none. A group with a NaN gets the scale NaN; infinities saturate.
//
// Append: key rows are the bf16 values of the rotation, correctly rounded: an error of the last bit next to a
// border would be a whole step of a code. FP32 decides wherever the value is farther from a bf16 border than
// its error bound; the others (about one in 2^11) are computed again in FP64.
//
// Both kernels are bound by memory (append: 128 bytes a head in, 128 or 36 out; read: 36 in, 128 out).
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

// Eight bf16 values (this lane's half of a group of 16; the other half is in lane ^ 1) to a word of codes.
// Returns the group's scale byte.
__device__ __forceinline__ uint32_t quantise8(const uint4& v, uint32_t& codes) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
  uint32_t top = 0;   // largest |x| as bits: a NaN is above infinity
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, max(u[i] & 0x7fffu, (u[i] >> 16) & 0x7fffu));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  // To four significant bits (the quotient of an 8-bit number and 6 is never close to a tie it is not).
  const float want = __fdiv_rn(__uint_as_float(top << 16), 6.0f);
  const uint32_t bits = __float_as_uint(want);
  uint32_t byte;
  if (want >= 6.103515625e-05f)   // 2^-14
    byte = ((bits + 0x7ffffu + ((bits >> 20) & 1u)) >> 20) - (112u << 3);
  else
    byte = static_cast<uint32_t>(__float2int_rn(want * 131072.0f));
  byte = min(byte, MAX_SCALE_BYTE);
  if (top > 0x7f80u) byte = 0xffu;
  const float scale = __half2float(__ushort_as_half(static_cast<unsigned short>(byte << 7)));
  const float inv = byte == 0 ? 0.0f : __frcp_rn(scale);
  codes = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float lo = __fadd_rn(__fadd_rn(bf16_lo(u[i]) * inv, 1536.0f), -1536.0f);
    const float hi = __fadd_rn(__fadd_rn(bf16_hi(u[i]) * inv, 1536.0f), -1536.0f);
    uint32_t two;
    asm("{\n\t.reg .b8 t, z;\n\t.reg .b16 q;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 t, %1, %2;\n\t"
        "mov.b16 q, {t, 0};\n\t"
        "cvt.u32.u16 %0, q;\n\t}"
        : "=r"(two)
        : "f"(hi), "f"(lo));
    codes |= two << (8 * i);
  }
  return byte;
}

// Stores a row's codes and scales; lane8 holds features 8 lane8 to 8 lane8 + 7 and its group's scale byte.
__device__ __forceinline__ void store_row(const View& c, int b, int h, int64_t pos, int lane8, bool ok,
                                          uint32_t codes, uint32_t byte) {
  uint32_t scales = (lane8 & 1) ? 0u : byte << (4 * lane8);
  scales |= __shfl_xor_sync(0xffffffffu, scales, 2);
  scales |= __shfl_xor_sync(0xffffffffu, scales, 4);
  if (!ok) return;
  uint8_t* block = c.p + b * c.sb + h * c.sh + (pos / BLOCK_ROWS) * c.sn;
  const int r = static_cast<int>(pos % BLOCK_ROWS);
  *reinterpret_cast<uint32_t*>(block + r * (HD / 2) + lane8 * 4) = codes;
  if (lane8 == 0) *reinterpret_cast<uint32_t*>(block + CODE_BYTES + r * GROUPS) = scales;
}

// ------------------------------------------------------------------------------- append

struct AppendParams {
  norm_rope::Common c;
  __nv_bfloat16* q_out;   // [B, Hq, T, 64]
  View cache[2];          // keys, values
  int64_t capacity;       // rows
};

// The correctly rounded bf16 values of a key row (up to FP64's own rounding).
template <bool NORM>
__device__ __forceinline__ uint4 key_row(const float (&x)[norm_rope::E], const float (&w)[norm_rope::E],
                                         const norm_rope::Turn& u, double eps) {
  using norm_rope::E;
  float r = 1.0f;
  if (NORM) r = norm_rope::inverse_rms(x, static_cast<float>(eps));
  uint32_t out[4];
  bool unsure = false;
#pragma unroll
  for (int i = 0; i < E / 2; ++i) {
    const float a = x[2 * i] * w[2 * i] * r, b = x[2 * i + 1] * w[2 * i + 1] * r;
    const float ac = a * u.c[i], bs = b * u.s[i], as = a * u.s[i], bc = b * u.c[i];
    const float y0 = ac - bs, y1 = as + bc;
    // In units of 2^-20 of the terms: rsqrtf .25, the sum of squares .35, six roundings .0625 each.
    const float e0 = (fabsf(ac) + fabsf(bs)) * 9.5367431640625e-07f;   // 2^-20
    const float e1 = (fabsf(as) + fabsf(bc)) * 9.5367431640625e-07f;
    out[i] = pack_bf16x2(y0 - e0, y1 - e1);
    unsure = unsure || out[i] != pack_bf16x2(y0 + e0, y1 + e1);
  }
  if (__any_sync(0xffffffffu, unsure)) {
    double rd = 1.0;
    if (NORM) {
      double ss = 0.0;
#pragma unroll
      for (int i = 0; i < E; ++i) ss += static_cast<double>(x[i]) * x[i];
#pragma unroll
      for (int m = 1; m < 8; m *= 2) ss += __shfl_xor_sync(0xffffffffu, ss, m);
      rd = 1.0 / sqrt(ss / HD + eps);
    }
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      const double a = x[2 * i] * rd * w[2 * i], b = x[2 * i + 1] * rd * w[2 * i + 1];
      const double c = u.c[i], s = u.s[i];
      out[i] = pack_bf16x2(static_cast<float>(a * c - b * s), static_cast<float>(a * s + b * c));
    }
  }
  return make_uint4(out[0], out[1], out[2], out[3]);
}

template <bool NORM>
__global__ void __launch_bounds__(norm_rope::THREADS)
    append_kernel(const __grid_constant__ AppendParams ap) {
  namespace nr = norm_rope;
  const nr::Common& p = ap.c;
  const int lane = threadIdx.x & 31, lane8 = lane & 7;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * nr::WARPS + (threadIdx.x >> 5);
  const int groups = (p.T + nr::ROWS - 1) / nr::ROWS;
  wait_for_previous_kernel();
  if (item >= static_cast<int64_t>(p.B) * groups * p.items_per_group) return;  // whole warps
  const int64_t bg = item / p.items_per_group;
  const int first = static_cast<int>(item % p.items_per_group) * p.heads_per_item;
  const int last = min(first + p.heads_per_item, p.Hq + 2 * p.Hkv);
  const int b = static_cast<int>(bg / groups);
  const int t = static_cast<int>(bg % groups) * nr::ROWS + (lane >> 3);
  const bool row = t < p.T;
  const int64_t pos = row ? nr::position_of(p, b, t) : 0;
  const bool ok = row && pos >= 0 && pos < p.table_len && pos < ap.capacity;
  if (row && !ok && lane8 == 0) atomicOr(&g_tt_status, TT_ERR_RANGE);
  nr::Turn u;
  nr::load_turn(p, ok ? pos : 0, lane8, u);
  const __nv_bfloat16* src = p.qkv + b * p.x_sb + static_cast<int64_t>(row ? t : 0) * p.x_st + lane8 * nr::E;
  float w[nr::E];
#pragma unroll
  for (int i = 0; i < nr::E; ++i) w[i] = 1.0f;
  int kind = -1;
#pragma unroll 2
  for (int h = first; h < last; ++h) {
    const int now = h < p.Hq ? 0 : h < p.Hq + p.Hkv ? 1 : 2;
    if (NORM && now != kind && now < 2) nr::load_weight(p, now, lane8, w);
    kind = now;
    uint4 v = *reinterpret_cast<const uint4*>(src + h * p.x_sh);
    float x[nr::E];
    if (now == 0) {
      float y[nr::E], r = 1.0f;
      nr::unpack8(v, x);
      if (NORM) r = nr::inverse_rms(x, static_cast<float>(p.eps));
      nr::turn_row(x, w, r, u, y);
      // A row whose position is outside the cache or the table is zero.
      const uint4 out = ok ? nr::pack8(y) : make_uint4(0, 0, 0, 0);
      if (row)
        *reinterpret_cast<uint4*>(ap.q_out + ((static_cast<int64_t>(b) * p.Hq + h) * p.T + t) * HD +
                                  lane8 * nr::E) = out;
      continue;
    }
    if (now == 1) {
      nr::unpack8(v, x);
      v = key_row<NORM>(x, w, u, p.eps);
    }
    uint32_t codes;
    const uint32_t byte = quantise8(v, codes);
    store_row(ap.cache[now - 1], b, h - p.Hq - (now - 1) * p.Hkv, pos, lane8, ok, codes, byte);
  }
}

// ------------------------------------------------------------------------------- read

struct ReadParams {
  View cache[2];
  __nv_bfloat16* out[2];          // [B, Hkv, rows, 64]
  int B, Hkv, rows;
  int64_t capacity;
  int64_t start;                  // first row where start_dev is NULL
  const int64_t* start_dev;       // first row of sequence b: start_dev[b * start_sb]
  int64_t start_sb;
};

constexpr int READ_THREADS = 256;
constexpr int READ_STEPS = 4;     // rows of a thread, so that as many loads are in flight

// Eight lanes a row: 4 bytes of codes and the group's scale each, 16 bytes out.
__global__ void __launch_bounds__(READ_THREADS) read_kernel(const __grid_constant__ ReadParams p) {
  const int lane8 = threadIdx.x & 7;
  wait_for_previous_kernel();
  const int64_t per_cache = static_cast<int64_t>(p.B) * p.Hkv * p.rows;
  constexpr int ROWS_PER_STEP = READ_THREADS / 8;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * (ROWS_PER_STEP * READ_STEPS) + (threadIdx.x >> 3);
  uint32_t codes[READ_STEPS], byte[READ_STEPS];
#pragma unroll
  for (int s = 0; s < READ_STEPS; ++s) {
    const int64_t at = base + s * ROWS_PER_STEP;
    codes[s] = byte[s] = 0;
    if (at >= 2 * per_cache) continue;
    const int kv = at >= per_cache ? 1 : 0;
    const int64_t rest = at - kv * per_cache;
    const int i = static_cast<int>(rest % p.rows);
    const int bh = static_cast<int>(rest / p.rows);
    const int b = bh / p.Hkv, h = bh - b * p.Hkv;
    const int64_t pos = (p.start_dev != nullptr ? p.start_dev[b * p.start_sb] : p.start) + i;
    if (pos < 0 || pos >= p.capacity) {   // reads as zero
      if (lane8 == 0) atomicOr(&g_tt_status, TT_ERR_RANGE);
      continue;
    }
    const View& c = p.cache[kv];
    const uint8_t* block = c.p + b * c.sb + h * c.sh + (pos / BLOCK_ROWS) * c.sn;
    const int r = static_cast<int>(pos % BLOCK_ROWS);
    codes[s] = *reinterpret_cast<const uint32_t*>(block + r * (HD / 2) + lane8 * 4);
    byte[s] = block[CODE_BYTES + r * GROUPS + (lane8 >> 1)];
  }
#pragma unroll
  for (int s = 0; s < READ_STEPS; ++s) {
    const int64_t at = base + s * ROWS_PER_STEP;
    if (at >= 2 * per_cache) continue;
    const int kv = at >= per_cache ? 1 : 0;
    uint32_t pairs[4], out[4];
    decode8(codes[s], pairs);
    const uint32_t scale = scale_pair(byte[s]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t y = mul_half2(pairs[i], scale);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&y));
      out[i] = pack_bf16x2(f.x, f.y);
    }
    *reinterpret_cast<uint4*>(p.out[kv] + (at - kv * per_cache) * HD + lane8 * 8) =
        make_uint4(out[0], out[1], out[2], out[3]);
  }
}

}  // namespace cache4
}  // namespace tt
