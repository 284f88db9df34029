// C-ABI implementation of the query/key norm and of the 4-bit KV cache (include/tt_attention.h): argument
// validation, variant choice and launches. Part of tt_attention_abi.cu, whose helpers (fail, prepare_device,
// check_launch, Launch, ...) and device status word it uses.
#pragma once

namespace {

// ------------------------------------------------------------------ query/key norm

struct NormRopeArgs {
  const void* qkv;
  const int64_t* strides;
  int64_t batch, q_len, q_heads, kv_heads;
  const void *q_weight, *k_weight;
  int weights_f32;
  const float *cos, *sin;
  int64_t table_len, position;
  const int64_t* position_dev;
  int64_t pos_sb, pos_st;
  double eps;
};

// Checks of what a pass over a projection has in common; `what` names the entry point.
tt_attn_status norm_rope_common(const std::string& what, const NormRopeArgs& a, tt::norm_rope::Common* c) {
  if (!a.qkv || !a.strides || !a.cos || !a.sin)
    return fail(TT_ATTN_BAD_ARG, what + ": qkv, its strides and the cos/sin tables must not be NULL");
  if (a.batch <= 0 || a.q_len <= 0 || a.q_heads <= 0 || a.kv_heads <= 0 || a.table_len <= 0)
    return fail(TT_ATTN_BAD_ARG, what + ": sizes must be positive");
  if ((a.q_weight == nullptr) != (a.k_weight == nullptr))
    return fail(TT_ATTN_BAD_ARG, what + ": both weights or neither");
  if (!(a.eps >= 0.0 && a.eps <= 3.0e38))
    return fail(TT_ATTN_BAD_ARG, what + ": eps must be finite and not negative");
  // (batch, 4 tokens, head) items, and q_len + position, stay far inside int32 / int64.
  constexpr int64_t kMax = INT32_MAX / 8;
  if (a.batch > kMax || a.q_len > kMax || a.q_heads > kMax || a.kv_heads > kMax ||
      (a.q_len + 3) / 4 > kMax / a.batch || a.q_heads + 2 * a.kv_heads > kMax / (a.batch * ((a.q_len + 3) / 4)))
    return fail(TT_ATTN_BAD_ARG, what + ": shape exceeds the supported CUDA grid limits");
  if (a.position_dev == nullptr && (a.position < 0 || a.position > a.table_len - a.q_len))
    return fail(TT_ATTN_BAD_ARG, what + ": position + q_len exceeds the cos/sin table");
  if (a.pos_sb < 0 || a.pos_st < 0)
    return fail(TT_ATTN_BAD_ARG, what + ": position strides must not be negative");
  if (reinterpret_cast<uintptr_t>(a.position_dev) % 8 != 0)
    return fail(TT_ATTN_BAD_ARG, what + ": the position must be 8-byte aligned");
  if (!aligned16(a.q_weight) || !aligned16(a.k_weight) || !aligned16(a.cos) || !aligned16(a.sin))
    return fail(TT_ATTN_BAD_ARG, what + ": the weights and the cos/sin tables must be 16-byte aligned");
  const int64_t size[3] = {a.batch, a.q_len, a.q_heads + 2 * a.kv_heads};
  for (int d = 0; d < 3; ++d)
    if (size[d] > 1 && (a.strides[d] <= 0 || a.strides[d] % 8 != 0))
      return fail(TT_ATTN_UNSUPPORTED, what + ": qkv needs strides in multiples of 8 elements; copy to "
                                              "contiguous storage first");
  if (!aligned16(a.qkv))
    return fail(TT_ATTN_UNSUPPORTED, what + ": qkv must be 16-byte aligned; copy to aligned storage first");
  c->qkv = static_cast<const __nv_bfloat16*>(a.qkv);
  c->x_sb = a.strides[0];
  c->x_st = a.strides[1];
  c->x_sh = a.strides[2];
  c->B = static_cast<int>(a.batch);
  c->T = static_cast<int>(a.q_len);
  c->Hq = static_cast<int>(a.q_heads);
  c->Hkv = static_cast<int>(a.kv_heads);
  c->w[0] = a.q_weight;
  c->w[1] = a.k_weight;
  c->w_f32 = a.weights_f32 != 0;
  c->cos = a.cos;
  c->sin = a.sin;
  c->table_len = a.table_len;
  c->position = a.position;
  c->position_dev = a.position_dev;
  c->pos_sb = a.pos_sb;
  c->pos_st = a.pos_st;
  c->eps = a.eps;
  return TT_ATTN_OK;
}

// Splits the heads of a group of four tokens into warp items: up to sixteen to an item, fewer where that leaves less than
// `warps` items. Returns the items.
int64_t norm_rope_items(tt::norm_rope::Common* c, bool values, int64_t warps) {
  const int64_t per_seq = (c->T + tt::norm_rope::ROWS - 1) / tt::norm_rope::ROWS, groups = c->B * per_seq;
  const int64_t heads = c->Hq + (values ? 2 : 1) * c->Hkv;
  const int per = static_cast<int>(
      std::max<int64_t>(1, std::min<int64_t>(tt::norm_rope::MAX_HEADS, groups * heads / warps)));
  c->per_item = per;
  c->items[0] = (c->Hq + per - 1) / per;
  c->items[1] = (c->Hkv + per - 1) / per;
  c->items[2] = values ? c->items[1] : 0;
  c->groups.set(static_cast<uint32_t>(per_seq));
  int64_t all = 0;
  for (int i = 0; i < 3; ++i) {
    c->each[i].set(static_cast<uint32_t>(std::max(1, c->items[i])));
    c->total[i] = static_cast<int>(groups * c->items[i]);
    all += c->total[i];
  }
  return all;
}

unsigned norm_rope_grid(int64_t items) {
  return static_cast<unsigned>((items + tt::norm_rope::WARPS - 1) / tt::norm_rope::WARPS);
}

constexpr int64_t kNormBackwardCtas = 5 * kPlanSms;   // but for rounding; its workspace has a row for each

// ------------------------------------------------------------------ 4-bit cache

// Byte strides of a cache [batch, kv_heads, blocks, 576]; those of size-1 dimensions do not matter.
bool cache4_view(void* base, const int64_t* st, int64_t batch, int64_t kv_heads, int64_t blocks,
                 tt::cache4::View* v) {
  constexpr int64_t row = tt::cache4::BLOCK_BYTES;
  const int64_t size[3] = {batch, kv_heads, blocks};
  int64_t s[3] = {st[0], st[1], st[2]};
  for (int d = 0; d < 3; ++d) {
    if (size[d] == 1) s[d] = row;
    if (s[d] < row || s[d] % 16 != 0) return false;
  }
  if (st[3] != 1) return false;
  *v = {static_cast<uint8_t*>(base), s[0], s[1], s[2]};
  return aligned16(base);
}

const char* const kCache4Layout =
    ": the caches need a unit last stride, others of at least 576 in multiples of 16 bytes and 16-byte aligned bases";

struct Cache4Dim {
  int64_t stride, size;
};

// Bytes from the first block to the end of the last one, or 0 where blocks might overlap: sorted by stride, each dimension
// has to step over all that lies inside it (as every layout does that slicing and transposing make).
template <size_t N>
int64_t cache4_extent(Cache4Dim (&&dims)[N]) {
  std::sort(dims, dims + N, [](const Cache4Dim& a, const Cache4Dim& b) { return a.stride < b.stride; });
  int64_t extent = tt::cache4::BLOCK_BYTES;
  for (const auto& [stride, size] : dims) {
    if (size == 1) continue;
    if (stride < extent || size - 1 > (INT64_MAX - extent) / stride) return 0;
    extent += (size - 1) * stride;
  }
  return extent;
}

// Caches that are written: no two blocks of the two may share a byte, as different warps write them. K and V may lie in one
// another's gaps where they have the same strides: their distance is one more dimension then.
tt_attn_status cache4_apart(const std::string& what, const tt::cache4::View (&c)[2], int64_t batch, int64_t kv_heads,
                            int64_t blocks) {
  int64_t extent[2];
  for (int i = 0; i < 2; ++i) {
    extent[i] = cache4_extent({{c[i].sb, batch}, {c[i].sh, kv_heads}, {c[i].sn, blocks}});
    if (extent[i] == 0)
      return fail(TT_ATTN_UNSUPPORTED, what + ": a cache's blocks must not overlap; each stride has to reach past the "
                                              "dimensions inside it");
  }
  const int first = c[0].p < c[1].p ? 0 : 1;
  const int64_t apart = c[1 - first].p - c[first].p;
  const bool alike = c[0].sb == c[1].sb && c[0].sh == c[1].sh && c[0].sn == c[1].sn;
  if (apart >= extent[first] ||
      (alike && cache4_extent({{apart, 2}, {c[0].sb, batch}, {c[0].sh, kv_heads}, {c[0].sn, blocks}}) != 0))
    return TT_ATTN_OK;
  return fail(TT_ATTN_BAD_ARG, what + ": the keys and the values need caches of their own, not over one another");
}

tt_attn_status cache4_sizes(const std::string& what, int64_t batch, int64_t kv_heads, int64_t blocks) {
  if (batch <= 0 || kv_heads <= 0 || blocks <= 0)
    return fail(TT_ATTN_BAD_ARG, what + ": sizes must be positive");
  if (blocks > INT32_MAX / (2 * tt::cache4::BLOCK_ROWS))
    return fail(TT_ATTN_BAD_ARG, what + ": the cache capacity must fit int32");
  return TT_ATTN_OK;
}

// Variant and split of one attention call over a 4-bit cache (sizes only: the workspace does not depend on the
// device).
struct Cache4Plan {
  int nt = 1;             // query rows of a tile, in eights
  int64_t row_tiles = 1;
  int cluster = 1;
  int64_t parts = 1;
  int64_t flat_ctas = 0;  // the flat kernel's CTAs; 0: the cluster kernel
};

// Measured (B200, us; cluster x parts, lengths half to all of the capacity, one query token):
//   flat / cluster: 768 units x 128 tiles 63 / 73; 512 x 64 27.9 / 28.7; 384 x 64 23.4 / 23.1; 128 x 64 14.1 / 10.2.
//   One K/V head, full lengths (near the copy rate): 4096 x 32 tiles 105 / 103, 16384 x 32 399 / 397; eight heads, 4096
//   sequences x 1 tile 62 / 144. More units than resident CTAs, whose starts then add up (one tile: full lengths): 12000 x 1
//   34 / 55; 2400 x 1 11.7 / 11.5; 2000 x 2 11.4 / 13.1; 1560 x 8 16.9 / 16.7; 1200 x 4 11.1 / 10.1. Sixteen-row tiles:
//   384 x 64 29.9 / 31.3; 1000 x 16 24.5 / 26.5; 256 x 32 18.8 / 20.2; 192 x 32 19.1 / 14.1; 256 x 16 17.0 / 15.9.
//   A unit's cluster, 96 units x 128 tiles: 1 to 8 CTAs 23.7, 16.7, 15.6, 13.2 (4), 14.5 (6), 14.7 (8); 256 x 64: 18.0,
//   17.0, 19.8, 19.2 (4): three CTAs to an SM are best, and two CTAs a unit where that leaves one.
//   Few units, parts without a cluster / clusters of 8 in one part or several: 12 x 64 tiles 5.0 / 4.1; 24 x 64 5.9 / 4.9;
//   4 x 256 5.3 / 5.9; 12 x 512 8.1 / 10.5; 8 x 512 7.1 / 8.6; 2 x 2048 12.1 / 8.1; 32 x 128 7.7 / 6.7.
constexpr int64_t kCache4FlatTiles = 24576, kCache4FlatTiles16 = 8000, kCache4FlatUnits = 12 * kPlanSms;

Cache4Plan cache4_plan(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t q_len, int64_t blocks) {
  namespace at = tt::cache4::attn;
  Cache4Plan pl;
  const int64_t rows = q_heads / kv_heads * q_len;
  pl.nt = rows <= 8 ? 1 : 2;
  pl.row_tiles = (rows + 8 * pl.nt - 1) / (8 * pl.nt);
  const int64_t units = batch * kv_heads * pl.row_tiles;
  const int64_t tiles = (blocks + at::TILE_BLOCKS - 1) / at::TILE_BLOCKS;
  // (The flat kernel counts tiles in 32 bits.)
  const bool flat = units >= kCache4FlatUnits || units * tiles > (pl.nt == 1 ? kCache4FlatTiles : kCache4FlatTiles16);
  if (flat && units >= kPlanSms && tiles <= INT32_MAX / units) {
    pl.flat_ctas = kPlanSms;
    return pl;
  }
  const int64_t most = (tiles + at::WARPS - 1) / at::WARPS;   // each warp with a tile at least
  const int64_t fill = std::max<int64_t>(3 * kPlanSms / units, units <= 2 * kPlanSms ? 2 : 1);
  if (units >= 32 || most <= 3 * at::MAX_CLUSTER) {
    pl.cluster = static_cast<int>(std::min<int64_t>({fill, most, at::MAX_CLUSTER}));
    return pl;
  }
  pl.parts = std::min<int64_t>({2 * kPlanSms / units, 32, most});
  if (most > 4 * pl.parts && 2 * kPlanSms / units > 32) {   // a long cache of a few heads
    pl.cluster = at::MAX_CLUSTER;
    pl.parts = 2 * kPlanSms / units / at::MAX_CLUSTER;
  }
  return pl;
}

int64_t cache4_flat_warps(const Cache4Plan& pl) {
  return pl.nt == 1 ? tt::cache4::attn::Flat<1>::WARPS : tt::cache4::attn::Flat<2>::WARPS;
}

// The flat kernel's table of units, in front of the records.
size_t cache4_table_bytes(const Cache4Plan& pl, int64_t units) {
  return pl.flat_ctas > 0 ? (static_cast<size_t>(units) * sizeof(int2) + 255) & ~size_t(255) : 0;
}

bool cache4_shape_ok(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t q_len, int64_t blocks) {
  constexpr int64_t kMax = INT32_MAX / (tt::cache4::MAX_QUERIES * tt::cache4::attn::MAX_CLUSTER);
  return batch > 0 && q_heads > 0 && kv_heads > 0 && q_len > 0 && blocks > 0 && q_heads % kv_heads == 0 &&
         q_len <= tt::cache4::MAX_QUERIES && blocks <= INT32_MAX / (2 * tt::cache4::BLOCK_ROWS) &&
         batch <= kMax && q_heads <= kMax / batch;
}

template <int NT, bool ONE>
cudaError_t launch_cache4(const Cache4Plan& pl, const tt::cache4::attn::Params& p, cudaStream_t stream) {
  namespace at = tt::cache4::attn;
  if (pl.flat_ctas > 0) {
    const Launch launch(dim3(static_cast<unsigned>(pl.flat_ctas)), at::Flat<NT>::WARPS * 32,
                        at::Flat<NT>::SMEM, 1, stream);
    cudaError_t e = cudaLaunchKernelEx(&launch.cfg, at::flat_kernel<NT, ONE>, p);
    if (e != cudaSuccess) return e;
    const int64_t rows = static_cast<int64_t>(p.B) * p.Hkv * p.G * p.T;
    const Launch merge(dim3(static_cast<unsigned>((rows + at::FLAT_COMBINE_WARPS - 1) / at::FLAT_COMBINE_WARPS)),
                       at::FLAT_COMBINE_WARPS * 32, 0, 1, stream);
    return cudaLaunchKernelEx(&merge.cfg, at::flat_combine_kernel, p, 8 * NT);
  }
  const int64_t grid = static_cast<int64_t>(p.B) * p.Hkv * pl.row_tiles * pl.parts * pl.cluster;
  const Launch launch(dim3(static_cast<unsigned>(grid)), at::THREADS, sizeof(at::Smem<NT>), pl.cluster, stream);
  cudaError_t e = cudaLaunchKernelEx(&launch.cfg, at::attention_kernel<NT, ONE>, p);
  if (e == cudaSuccess && pl.parts > 1) {
    const Launch merge(dim3(static_cast<unsigned>(static_cast<int64_t>(p.B) * p.Hkv * p.G * p.T)),
                       at::COMBINE_WARPS * 32, 0, 1, stream);
    e = cudaLaunchKernelEx(&merge.cfg, at::combine_kernel, p, 8 * NT);
  }
  return e;
}

tt_attn_status set_cache4_attributes(int dev) {
  namespace at = tt::cache4::attn;
  static std::atomic<bool> done[kMaxDevices] = {};
  if (done[dev].load(std::memory_order_acquire)) return TT_ATTN_OK;
  cudaError_t e = cudaSuccess;
  for (auto fn : {at::attention_kernel<1, true>, at::attention_kernel<1, false>})
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               static_cast<int>(sizeof(at::Smem<1>)));
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(at::attention_kernel<2, false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(sizeof(at::Smem<2>)));
  for (auto fn : {at::flat_kernel<1, true>, at::flat_kernel<1, false>})
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               static_cast<int>(at::Flat<1>::SMEM));
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(at::flat_kernel<2, false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(at::Flat<2>::SMEM));
  if (e != cudaSuccess) return cuda_fail("cudaFuncSetAttribute", e);
  done[dev].store(true, std::memory_order_release);
  return TT_ATTN_OK;
}

}  // namespace

extern "C" {

TT_ATTN_API tt_attn_status tt_attn_qkv_norm_rope_bf16(
    const void* qkv, const int64_t* qkv_strides, int64_t batch, int64_t q_len, int64_t q_heads,
    int64_t kv_heads, const void* q_weight, const void* k_weight, int weights_f32, const float* cos,
    const float* sin, int64_t table_len, int64_t position, const int64_t* position_dev,
    int64_t position_sb, int64_t position_st, double eps, void* q_out, void* k_out, void* stream) {
  namespace nr = tt::norm_rope;
  nr::ForwardParams p{};
  tt_attn_status st = norm_rope_common(
      "qkv_norm_rope",
      {qkv, qkv_strides, batch, q_len, q_heads, kv_heads, q_weight, k_weight, weights_f32, cos, sin, table_len,
       position, position_dev, position_sb, position_st, eps},
      &p.c);
  if (st != TT_ATTN_OK) return st;
  if (!q_out || !k_out || !aligned16(q_out) || !aligned16(k_out))
    return fail(TT_ATTN_BAD_ARG, "qkv_norm_rope: the outputs must not be NULL and be 16-byte aligned");
  int dev = 0;
  if ((st = prepare_device(&dev)) != TT_ATTN_OK) return st;
  p.out[0] = static_cast<__nv_bfloat16*>(q_out);
  p.out[1] = static_cast<__nv_bfloat16*>(k_out);
  const int64_t items = norm_rope_items(&p.c, false, 16 * kPlanSms);
  const Launch launch(dim3(norm_rope_grid(items)), nr::THREADS, 0, 1, static_cast<cudaStream_t>(stream));
  const cudaError_t le = q_weight != nullptr ? cudaLaunchKernelEx(&launch.cfg, nr::forward_kernel<true>, p)
                                             : cudaLaunchKernelEx(&launch.cfg, nr::forward_kernel<false>, p);
  return check_launch("qkv_norm_rope launch", le);
}

TT_ATTN_API size_t tt_attn_qkv_norm_rope_backward_workspace_size(void) {
  return static_cast<size_t>(kNormBackwardCtas + 2) * TT_ATTN_HEAD_DIM * sizeof(float);
}

TT_ATTN_API tt_attn_status tt_attn_qkv_norm_rope_backward_bf16(
    const void* qkv, const int64_t* qkv_strides, int64_t batch, int64_t q_len, int64_t q_heads,
    int64_t kv_heads, const void* q_weight, const void* k_weight, int weights_f32, const float* cos,
    const float* sin, int64_t table_len, int64_t position, const int64_t* position_dev,
    int64_t position_sb, int64_t position_st, double eps, const void* dq, const int64_t* dq_strides,
    const void* dk, const int64_t* dk_strides, const void* dv, const int64_t* dv_strides, void* dqkv,
    void* dq_weight, void* dk_weight, void* workspace, size_t workspace_bytes, void* stream) {
  namespace nr = tt::norm_rope;
  nr::BackwardParams p{};
  tt_attn_status st = norm_rope_common(
      "qkv_norm_rope backward",
      {qkv, qkv_strides, batch, q_len, q_heads, kv_heads, q_weight, k_weight, weights_f32, cos, sin, table_len,
       position, position_dev, position_sb, position_st, eps},
      &p.c);
  if (st != TT_ATTN_OK) return st;
  const bool norm = q_weight != nullptr;
  if (!dqkv || !aligned16(dqkv))
    return fail(TT_ATTN_BAD_ARG, "qkv_norm_rope backward: dqkv must not be NULL and be 16-byte aligned");
  if (norm && (!dq_weight || !dk_weight || !workspace || !aligned16(workspace) ||
               workspace_bytes < tt_attn_qkv_norm_rope_backward_workspace_size()))
    return fail(TT_ATTN_BAD_ARG, "qkv_norm_rope backward: the weights' gradients must not be NULL, and workspace "
                                 "tt_attn_qkv_norm_rope_backward_workspace_size() bytes, 16-byte aligned");
  for (const void* w : {static_cast<const void*>(dq_weight), static_cast<const void*>(dk_weight)})
    if (norm && reinterpret_cast<uintptr_t>(w) % (weights_f32 ? 4 : 2) != 0)
      return fail(TT_ATTN_BAD_ARG, "qkv_norm_rope backward: the weights' gradients must be aligned to their type");
  const void* g[3] = {dq, dk, dv};
  const int64_t* gs[3] = {dq_strides, dk_strides, dv_strides};
  for (int i = 0; i < 3; ++i) {
    if (g[i] == nullptr) continue;
    if (gs[i] == nullptr)
      return fail(TT_ATTN_BAD_ARG, "qkv_norm_rope backward: a gradient needs its strides");
    const Shape4 s = canonical(batch, i == 0 ? q_heads : kv_heads, q_len, gs[i]);
    if (!aligned16(g[i]) || !strides_ok(s.stride))
      return fail(TT_ATTN_UNSUPPORTED,
                  "qkv_norm_rope backward: gradients need a unit last stride, other strides in multiples of 8 "
                  "elements and 16-byte aligned bases; copy to aligned contiguous storage first");
    p.g[i] = static_cast<const __nv_bfloat16*>(g[i]);
    p.g_sb[i] = s.stride[0];
    p.g_sh[i] = s.stride[1];
    p.g_st[i] = s.stride[2];
  }
  int dev = 0;
  if ((st = prepare_device(&dev)) != TT_ATTN_OK) return st;
  p.dx = static_cast<__nv_bfloat16*>(dqkv);
  p.partial = static_cast<float*>(workspace);
  p.dw[0] = dq_weight;
  p.dw[1] = dk_weight;
  // CTAs for each kind of heads in proportion to what they read and write: x, dy and dx, or dv twice.
  norm_rope_items(&p.c, true, 16 * kPlanSms);
  const int64_t weight[3] = {3 * q_heads, 3 * kv_heads, 2 * kv_heads}, sum = weight[0] + weight[1] + weight[2];
  int64_t blocks = 0;
  for (int i = 0; i < 3; ++i) {
    p.ctas[i] = static_cast<int>(std::max<int64_t>(
        1, std::min<int64_t>(norm_rope_grid(p.c.total[i]), kNormBackwardCtas * weight[i] / sum)));
    blocks += p.ctas[i];
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const Launch launch(dim3(static_cast<unsigned>(blocks)), nr::THREADS, 0, 1, s);
  cudaError_t le = norm ? cudaLaunchKernelEx(&launch.cfg, nr::backward_kernel<true>, p)
                        : cudaLaunchKernelEx(&launch.cfg, nr::backward_kernel<false>, p);
  if (le == cudaSuccess && norm) {
    const Launch reduce(dim3(2 * nr::HD / nr::REDUCE_FEATURES), nr::REDUCE_THREADS * nr::REDUCE_FEATURES, 0, 1, s);
    le = cudaLaunchKernelEx(&reduce.cfg, nr::reduce_kernel, p);
  }
  return check_launch("qkv_norm_rope backward launch", le);
}

TT_ATTN_API tt_attn_status tt_attn_cache4_append_bf16(
    const void* qkv, const int64_t* qkv_strides, int64_t batch, int64_t q_len, int64_t q_heads,
    int64_t kv_heads, const void* q_weight, const void* k_weight, int weights_f32, const float* cos,
    const float* sin, int64_t table_len, int64_t position, const int64_t* position_dev,
    int64_t position_sb, double eps, void* q_out, void* cache_k, const int64_t* ck_strides,
    void* cache_v, const int64_t* cv_strides, int64_t blocks, void* stream) {
  namespace nr = tt::norm_rope;
  namespace c4 = tt::cache4;
  c4::AppendParams p{};
  tt_attn_status st = norm_rope_common(
      "cache4_append",
      {qkv, qkv_strides, batch, q_len, q_heads, kv_heads, q_weight, k_weight, weights_f32, cos, sin, table_len,
       position, position_dev, position_sb, 0, eps},
      &p.c);
  if (st != TT_ATTN_OK) return st;
  if ((st = cache4_sizes("cache4_append", batch, kv_heads, blocks)) != TT_ATTN_OK) return st;
  if (!q_out || !aligned16(q_out) || !cache_k || !cache_v || !ck_strides || !cv_strides)
    return fail(TT_ATTN_BAD_ARG, "cache4_append: q_out, the caches and their strides must not be NULL, and q_out "
                                 "16-byte aligned");
  if (!cache4_view(cache_k, ck_strides, batch, kv_heads, blocks, &p.cache[0]) ||
      !cache4_view(cache_v, cv_strides, batch, kv_heads, blocks, &p.cache[1]))
    return fail(TT_ATTN_UNSUPPORTED, std::string("cache4_append") + kCache4Layout);
  p.capacity = blocks * c4::BLOCK_ROWS;
  if (position_dev == nullptr && position > p.capacity - q_len)
    return fail(TT_ATTN_BAD_ARG, "cache4_append: position + q_len exceeds the cache capacity");
  if ((st = cache4_apart("cache4_append", p.cache, batch, kv_heads, blocks)) != TT_ATTN_OK) return st;
  int dev = 0;
  if ((st = prepare_device(&dev)) != TT_ATTN_OK) return st;
  p.q_out = static_cast<__nv_bfloat16*>(q_out);
  const int64_t items = norm_rope_items(&p.c, true, 16 * kPlanSms);
  const Launch launch(dim3(norm_rope_grid(items)), nr::THREADS, 0, 1, static_cast<cudaStream_t>(stream));
  const cudaError_t le = q_weight != nullptr ? cudaLaunchKernelEx(&launch.cfg, c4::append_kernel<true>, p)
                                             : cudaLaunchKernelEx(&launch.cfg, c4::append_kernel<false>, p);
  return check_launch("cache4_append launch", le);
}

TT_ATTN_API tt_attn_status tt_attn_cache4_read_bf16(
    const void* cache_k, const int64_t* ck_strides, const void* cache_v, const int64_t* cv_strides,
    int64_t batch, int64_t kv_heads, int64_t blocks, int64_t start, const int64_t* start_dev,
    int64_t start_sb, int64_t rows, void* k_out, void* v_out, void* stream) {
  namespace c4 = tt::cache4;
  c4::ReadParams p{};
  tt_attn_status st = cache4_sizes("cache4_read", batch, kv_heads, blocks);
  if (st != TT_ATTN_OK) return st;
  if (!cache_k || !cache_v || !ck_strides || !cv_strides || !k_out || !v_out || !aligned16(k_out) ||
      !aligned16(v_out))
    return fail(TT_ATTN_BAD_ARG, "cache4_read: the caches, their strides and the outputs must not be NULL, and the "
                                 "outputs 16-byte aligned");
  if (rows <= 0) return fail(TT_ATTN_BAD_ARG, "cache4_read: sizes must be positive");
  constexpr int64_t kMax = INT32_MAX / 8;
  const int64_t chunks = rows / c4::READ_ROWS + 1;
  if (batch > kMax || kv_heads > kMax / batch || rows > INT32_MAX / 2 || chunks > kMax / (batch * kv_heads))
    return fail(TT_ATTN_BAD_ARG, "cache4_read: shape exceeds the supported CUDA grid limits");
  if (start_sb < 0 || reinterpret_cast<uintptr_t>(start_dev) % 8 != 0)
    return fail(TT_ATTN_BAD_ARG, "cache4_read: the start needs a stride that is not negative and 8-byte alignment");
  if (!cache4_view(const_cast<void*>(cache_k), ck_strides, batch, kv_heads, blocks, &p.cache[0]) ||
      !cache4_view(const_cast<void*>(cache_v), cv_strides, batch, kv_heads, blocks, &p.cache[1]))
    return fail(TT_ATTN_UNSUPPORTED, std::string("cache4_read") + kCache4Layout);
  p.capacity = blocks * c4::BLOCK_ROWS;
  if (start_dev == nullptr && (start < 0 || start > p.capacity - rows))
    return fail(TT_ATTN_BAD_ARG, "cache4_read: start + rows exceeds the cache capacity");
  int dev = 0;
  if ((st = prepare_device(&dev)) != TT_ATTN_OK) return st;
  p.out[0] = static_cast<__nv_bfloat16*>(k_out);
  p.out[1] = static_cast<__nv_bfloat16*>(v_out);
  p.B = static_cast<int>(batch);
  p.Hkv = static_cast<int>(kv_heads);
  p.rows = static_cast<int>(rows);
  p.start = start;
  p.start_dev = start_dev;
  p.start_sb = start_sb;
  p.chunks.set(static_cast<uint32_t>((rows + c4::READ_ROWS - 1) / c4::READ_ROWS));
  p.heads.set(static_cast<uint32_t>(kv_heads));
  const int64_t items = 2 * batch * kv_heads * p.chunks.d;
  const Launch launch(dim3(static_cast<unsigned>((items + c4::READ_WARPS - 1) / c4::READ_WARPS)),
                      c4::READ_WARPS * 32, 0, 1, static_cast<cudaStream_t>(stream));
  return check_launch("cache4_read launch", cudaLaunchKernelEx(&launch.cfg, c4::read_kernel, p));
}

TT_ATTN_API size_t tt_attn_cache4_workspace_size(int64_t batch, int64_t q_heads, int64_t kv_heads,
                                                 int64_t q_len, int64_t blocks) {
  if (!cache4_shape_ok(batch, q_heads, kv_heads, q_len, blocks)) return 0;
  const Cache4Plan pl = cache4_plan(batch, q_heads, kv_heads, q_len, blocks);
  const int64_t units = batch * kv_heads * pl.row_tiles;
  if (pl.flat_ctas == 0 && pl.parts == 1) return 0;
  const int64_t slots = pl.flat_ctas > 0 ? units + pl.flat_ctas * cache4_flat_warps(pl) : units * pl.parts;
  return cache4_table_bytes(pl, units) + static_cast<size_t>(slots) * 8 * pl.nt *
         tt::cache4::attn::REC * sizeof(float);
}

TT_ATTN_API tt_attn_status tt_attn_cache4_forward_bf16(
    const void* q, const int64_t* q_strides, const void* cache_k, const int64_t* ck_strides,
    const void* cache_v, const int64_t* cv_strides, int64_t batch, int64_t q_heads, int64_t kv_heads,
    int64_t q_len, int64_t blocks, int64_t head_dim, const int32_t* kv_lens, void* out, float* lse,
    void* workspace, size_t workspace_bytes, void* stream) {
  namespace at = tt::cache4::attn;
  if (!q || !q_strides || !cache_k || !ck_strides || !cache_v || !cv_strides || !out)
    return fail(TT_ATTN_BAD_ARG, "cache4_attention: q, the caches, out and the stride arrays must not be NULL");
  if (head_dim != TT_ATTN_HEAD_DIM)
    return fail(TT_ATTN_BAD_ARG, "cache4_attention currently supports only head_dim=64");
  tt_attn_status st = cache4_sizes("cache4_attention", batch, kv_heads, blocks);
  if (st != TT_ATTN_OK) return st;
  if (q_heads <= 0 || q_len <= 0) return fail(TT_ATTN_BAD_ARG, "cache4_attention: sizes must be positive");
  if (q_heads % kv_heads != 0)
    return fail(TT_ATTN_BAD_ARG, "cache4_attention: q heads must be a multiple of the K/V heads");
  if (q_len > TT_ATTN_CACHE4_MAX_QUERIES)
    return fail(TT_ATTN_BAD_ARG, "cache4_attention: at most 16 query tokens");
  if (!cache4_shape_ok(batch, q_heads, kv_heads, q_len, blocks))
    return fail(TT_ATTN_BAD_ARG, "cache4_attention: shape exceeds the supported CUDA grid limits");
  const Shape4 qs = canonical(batch, q_heads, q_len, q_strides);
  at::Params p{};
  if (!operand_ok(q, qs))
    return fail(TT_ATTN_UNSUPPORTED, "cache4_attention: q needs a unit last stride, other strides in multiples of "
                                     "8 elements and a 16-byte aligned base; copy to aligned contiguous storage first");
  if (!cache4_view(const_cast<void*>(cache_k), ck_strides, batch, kv_heads, blocks, &p.cache[0]) ||
      !cache4_view(const_cast<void*>(cache_v), cv_strides, batch, kv_heads, blocks, &p.cache[1]))
    return fail(TT_ATTN_UNSUPPORTED, std::string("cache4_attention") + kCache4Layout);
  if (!aligned16(out)) return fail(TT_ATTN_BAD_ARG, "cache4_attention: out must be 16-byte aligned");
  for (const void* ptr : {static_cast<const void*>(kv_lens), static_cast<const void*>(lse)})
    if (reinterpret_cast<uintptr_t>(ptr) % 4 != 0)
      return fail(TT_ATTN_BAD_ARG, "cache4_attention: kv_lens and lse must be 4-byte aligned");
  const size_t need = tt_attn_cache4_workspace_size(batch, q_heads, kv_heads, q_len, blocks);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned16(workspace)))
    return fail(TT_ATTN_BAD_ARG, "cache4_attention: workspace is smaller than tt_attn_cache4_workspace_size() or "
                                 "not 16-byte aligned");
  int dev = 0;
  if ((st = prepare_device(&dev)) != TT_ATTN_OK) return st;
  if ((st = set_cache4_attributes(dev)) != TT_ATTN_OK) return st;
  const Cache4Plan pl = cache4_plan(batch, q_heads, kv_heads, q_len, blocks);
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_sb = qs.stride[0];
  p.q_sh = qs.stride[1];
  p.q_st = qs.stride[2];
  p.lens = kv_lens;
  p.B = static_cast<int>(batch);
  p.Hkv = static_cast<int>(kv_heads);
  p.G = static_cast<int>(q_heads / kv_heads);
  p.T = static_cast<int>(q_len);
  p.row_tiles = static_cast<int>(pl.row_tiles);
  p.blocks = static_cast<int>(blocks);
  p.cluster = pl.cluster;
  p.parts = static_cast<int>(pl.parts);
  p.o = static_cast<__nv_bfloat16*>(out);
  p.lse = lse;
  p.parts_of = static_cast<int2*>(workspace);
  p.records = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) +
                                       cache4_table_bytes(pl, batch * kv_heads * pl.row_tiles));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return check_launch("cache4_attention launch",
                      pl.nt == 2                  ? launch_cache4<2, false>(pl, p, s)
                      : q_heads * q_len == kv_heads ? launch_cache4<1, true>(pl, p, s)
                                                    : launch_cache4<1, false>(pl, p, s));
}

}  // extern "C"
