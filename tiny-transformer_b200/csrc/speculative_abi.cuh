// C-ABI implementation of the speculative-decoding operators (include/tt_attention.h): argument
// validation, variant choice and launches. Part of tt_attention_abi.cu, whose helpers (fail,
// prepare_device, encode_map, ...) and device status word it uses.
#pragma once

namespace {

// Variant and split of one tree-attention call (sizes only: the workspace does not depend on the
// device).
struct TreePlan {
  bool persistent = false;
  int64_t rows = 0;       // query rows of a CTA's tile
  int64_t row_tiles = 1;  // tiles of one (batch, K/V head)
  int splits = 1;         // cluster kernel: CTAs per cluster
  int dup = 1;            // persistent kernel: copies of the rows in a 128-row tile
  int64_t grid = 0;       // persistent kernel: CTAs
  bool whole = false;     // persistent kernel: no unit is shared by CTAs
};

TreePlan tree_plan(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t nodes,
                   int64_t capacity) {
  TreePlan pl;
  const int64_t rows = q_heads / kv_heads * nodes;
  const int64_t tree_tiles = (nodes + tt::tree::KEYS - 1) / tt::tree::KEYS;
  const int64_t tiles = tree_tiles + (capacity + tt::tree::KEYS - 1) / tt::tree::KEYS;
  // The cluster kernel reads the cache once per 16 rows, but starts and ends in half the persistent
  // kernel's time. With one row tile it always wins (142 against 165 us for 16 rows at B = 64, 1024-
  // 8192 cached); with more, up to about 8192 tile reads (us persistent / cluster: 96 sequences, 32
  // rows, capacity 2048, 3072 reads 19.6 / 16.8; 384, 32, 1024, 6144 reads 33.6 / 28.8; 96, 24, 8192,
  // 12288 reads 30.9 / 40.1; 384, 32, 4096, 24576 reads 60 / 71).
  const int64_t cluster_tiles = (rows + tt::tree::ROWS - 1) / tt::tree::ROWS;
  const int64_t reads = batch * kv_heads * cluster_tiles * (tiles - tree_tiles);
  pl.persistent = nodes > tt::tree::CLUSTER_NODES || (cluster_tiles > 1 && reads > 8192);
  if (pl.persistent) {
    constexpr int64_t bm = tt::tree::persist::BM;
    pl.row_tiles = (rows + bm - 1) / bm;
    pl.rows = (rows + pl.row_tiles - 1) / pl.row_tiles;
    pl.dup = pl.rows <= bm / 4 ? 4 : pl.rows <= bm / 2 ? 2 : 1;
    // Sharing a unit costs a second epilogue and the merge kernel, about eight tiles' time.
    const int64_t units = batch * kv_heads * pl.row_tiles;
    pl.whole = tiles <= 9;
    pl.grid = std::min<int64_t>(kPlanSms, pl.whole ? units : units * tiles);
    return pl;
  }
  // Three CTAs fit an SM; a cluster shares a sequence's tiles: enough CTAs to fill the SMs once, and
  // for long caches CTAs of about 16 tiles whatever their number, so that the last ones to run are
  // short (us at 1, 2, 3, 4 CTAs a sequence: 384 sequences x 64 tiles 87, 83, 81, 82; 768 x 32 tiles
  // 86, 84, 87, 92; 768 x 8 tiles 30, 37, 47, 54; 96 x 16 tiles 16, 12, 11, 10.4).
  pl.rows = tt::tree::ROWS;
  pl.row_tiles = cluster_tiles;
  const int64_t units = batch * kv_heads * pl.row_tiles, cached = tiles - tree_tiles;
  const int64_t fill = std::min<int64_t>({tt::tree::MAX_SPLITS, cached, 3 * kPlanSms / units});
  pl.splits = static_cast<int>(std::max<int64_t>({1, fill, std::min<int64_t>(3, cached / 16)}));
  return pl;
}

size_t tree_starts_bytes(const TreePlan& pl) {
  return (static_cast<size_t>(pl.grid) * sizeof(tt::tree::persist::Start) + 255) & ~size_t(255);
}

bool tree_shape_ok(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t nodes,
                   int64_t capacity) {
  const int64_t max_rows = INT32_MAX / (TT_ATTN_TREE_MAX_NODES * tt::tree::MAX_SPLITS);
  return batch > 0 && q_heads > 0 && kv_heads > 0 && nodes > 0 && capacity > 0 &&
         q_heads % kv_heads == 0 && nodes <= TT_ATTN_TREE_MAX_NODES &&
         capacity <= INT32_MAX - tt::tree::KEYS && batch <= max_rows && q_heads <= max_rows &&
         batch <= max_rows / q_heads &&
         // cost (key tiles and the fixed part) of all (batch, q head, 128-row tile): the persistent
         // kernel counts it in 32 bits
         (capacity / tt::tree::KEYS + 1 + TT_ATTN_TREE_MAX_NODES / tt::tree::KEYS +
          tt::tree::persist::UNIT_COST) * 2 <= INT32_MAX / (batch * q_heads);
}

// Shared memory beyond the default 48 KiB, for the kernels that may ask for it.
tt_attn_status set_speculative_attributes(int dev) {
  static std::atomic<bool> done[kMaxDevices] = {};
  cudaError_t e = cudaSuccess;
  if (!done[dev].load(std::memory_order_acquire)) {
    for (auto fn : {tt::tree::tree_attention_kernel<false>, tt::tree::tree_attention_kernel<true>})
      if (e == cudaSuccess)
        e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 static_cast<int>(tt::tree::kSmemBytes));
    for (auto fn : {tt::tree::persist::tree_persistent_kernel<1>,
                    tt::tree::persist::tree_persistent_kernel<2>,
                    tt::tree::persist::tree_persistent_kernel<4>})
      if (e == cudaSuccess)
        e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 static_cast<int>(tt::tree::persist::kSmemBytes));
    for (auto fn : {tt::verify::tree_verify_kernel<false, false>,
                    tt::verify::tree_verify_kernel<false, true>,
                    tt::verify::tree_verify_kernel<true, false>,
                    tt::verify::tree_verify_kernel<true, true>})
      if (e == cudaSuccess)
        e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 static_cast<int>(tt::verify::kMaxDynamicSmem));
    if (e == cudaSuccess) done[dev].store(true, std::memory_order_release);
  }
  if (e != cudaSuccess)
    return cuda_fail("cudaFuncSetAttribute", e);
  return TT_ATTN_OK;
}

// Launch configuration of the speculative operators: a cluster size (1: none), and a programmatic
// launch, so that a kernel's launch and prologue run under the end of the kernel before it (every
// one of these kernels waits for that kernel on the device before it touches memory; 0.5 to 1.5 us
// a call on the smallest ones).
struct Launch {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  Launch(dim3 grid, int threads, size_t smem, int cluster, cudaStream_t stream) {
    cfg.gridDim = grid;
    cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
  }
};

tt_attn_status launch_tree_persistent(const TreePlan& pl, const tt::tree::Params& tp,
                                      void* workspace,
                                      int sm_count, const CUtensorMap& tmk, const CUtensorMap& tmv,
                                      const CUtensorMap& tmtk, const CUtensorMap& tmtv,
                                      cudaStream_t stream) {
  namespace ps = tt::tree::persist;
  ps::Params p{};
  p.t = tp;
  p.rows = static_cast<int>(pl.rows);
  p.units = static_cast<int>(tp.Hkv * pl.row_tiles);
  p.tree_tiles = (tp.N + tt::tree::KEYS - 1) / tt::tree::KEYS;
  p.whole = pl.whole;
  p.starts = static_cast<ps::Start*>(workspace);
  p.records = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + tree_starts_bytes(pl));
  const int grid = static_cast<int>(std::min<int64_t>(pl.grid, sm_count > 0 ? sm_count : kPlanSms));
  auto kernel = pl.dup == 4 ? ps::tree_persistent_kernel<4>
                            : pl.dup == 2 ? ps::tree_persistent_kernel<2>
                                          : ps::tree_persistent_kernel<1>;
  const Launch main(dim3(static_cast<unsigned>(grid)), ps::THREADS, ps::kSmemBytes, 1, stream);
  cudaError_t le = cudaLaunchKernelEx(&main.cfg, kernel, tmk, tmv, tmtk, tmtv, p);
  if (le == cudaSuccess && grid > 1 && !pl.whole) {
    const Launch merge(dim3(static_cast<unsigned>(grid - 1),
                            static_cast<unsigned>((pl.rows + ps::COMBINE_ROWS - 1) / ps::COMBINE_ROWS)),
                       ps::COMBINE_THREADS, 0, 1, stream);
    le = cudaLaunchKernelEx(&merge.cfg, ps::tree_combine_kernel, p, grid);
  }
  return check_launch("tree_persistent_kernel launch", le);
}

// [batch, heads, rows, 64] operand of the speculative operators: readable in place?
bool operand_ok(const void* p, const Shape4& s) { return aligned16(p) && strides_ok(s.stride); }

}  // namespace

extern "C" {

TT_ATTN_API size_t tt_attn_tree_workspace_size(int64_t batch, int64_t q_heads, int64_t kv_heads,
                                               int64_t nodes, int64_t capacity) {
  if (!tree_shape_ok(batch, q_heads, kv_heads, nodes, capacity)) return 0;
  const TreePlan pl = tree_plan(batch, q_heads, kv_heads, nodes, capacity);
  if (!pl.persistent) return 0;
  return tree_starts_bytes(pl) +
         (pl.whole ? 0 : static_cast<size_t>(pl.grid) * 2 * pl.rows * tt::tree::REC * sizeof(float));
}

TT_ATTN_API tt_attn_status tt_attn_tree_forward_bf16(
    const void* q, const int64_t* q_strides, const void* tree_k, const int64_t* tk_strides,
    const void* tree_v, const int64_t* tv_strides, const void* cache_k, const int64_t* ck_strides,
    const void* cache_v, const int64_t* cv_strides, int64_t batch, int64_t q_heads,
    int64_t kv_heads, int64_t nodes, int64_t capacity, int64_t head_dim, const int32_t* parents,
    int64_t parents_stride, const int32_t* cache_lens, void* out, float* lse, void* workspace,
    size_t workspace_bytes, void* stream) {
  namespace tr = tt::tree;
  // ---- validation: everything is checked before any CUDA call
  if (!q || !tree_k || !tree_v || !cache_k || !cache_v || !parents || !out || !q_strides ||
      !tk_strides || !tv_strides || !ck_strides || !cv_strides)
    return fail(TT_ATTN_BAD_ARG, "tree_attention: q, the tree's and the cache's K/V, parents, out "
                                 "and the stride arrays must not be NULL");
  if (head_dim != TT_ATTN_HEAD_DIM)
    return fail(TT_ATTN_BAD_ARG, "tree_attention currently supports only head_dim=64");
  if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || nodes <= 0 || capacity <= 0)
    return fail(TT_ATTN_BAD_ARG,
                "tree_attention: batch, heads, nodes and cache capacity must be positive");
  if (q_heads % kv_heads != 0)
    return fail(TT_ATTN_BAD_ARG, "tree_attention: q heads must be a multiple of the K/V heads");
  if (nodes > TT_ATTN_TREE_MAX_NODES)
    return fail(TT_ATTN_BAD_ARG, "tree_attention: at most 256 nodes per tree");
  if (capacity > INT32_MAX - tr::KEYS)
    return fail(TT_ATTN_BAD_ARG, "tree_attention: the cache capacity must fit int32");
  if (parents_stride != 0 && parents_stride < nodes)
    return fail(TT_ATTN_BAD_ARG, "tree_attention: parents_stride must be 0 or at least nodes");
  if (!tree_shape_ok(batch, q_heads, kv_heads, nodes, capacity))
    return fail(TT_ATTN_BAD_ARG, "tree_attention: shape exceeds the supported CUDA grid limits");
  const Shape4 qs = canonical(batch, q_heads, nodes, q_strides);
  const Shape4 tks = canonical(batch, kv_heads, nodes, tk_strides);
  const Shape4 tvs = canonical(batch, kv_heads, nodes, tv_strides);
  const Shape4 cks = canonical(batch, kv_heads, capacity, ck_strides);
  const Shape4 cvs = canonical(batch, kv_heads, capacity, cv_strides);
  if (!operand_ok(q, qs) || !operand_ok(tree_k, tks) || !operand_ok(tree_v, tvs) ||
      !operand_ok(cache_k, cks) || !operand_ok(cache_v, cvs))
    return fail(TT_ATTN_UNSUPPORTED,
                "tree_attention: q and the K/V tensors need a unit last stride, other strides in "
                "multiples of 8 elements and 16-byte aligned bases; copy to aligned contiguous "
                "storage first");
  if (!aligned16(out)) return fail(TT_ATTN_BAD_ARG, "tree_attention: out must be 16-byte aligned");
  for (const void* ptr : {static_cast<const void*>(parents), static_cast<const void*>(cache_lens),
                          static_cast<const void*>(lse)})
    if (reinterpret_cast<uintptr_t>(ptr) % 4 != 0)
      return fail(TT_ATTN_BAD_ARG, "tree_attention: parents, cache_lens and lse must be 4-byte aligned");
  const size_t need = tt_attn_tree_workspace_size(batch, q_heads, kv_heads, nodes, capacity);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned16(workspace)))
    return fail(TT_ATTN_BAD_ARG, "tree_attention: workspace is smaller than "
                                 "tt_attn_tree_workspace_size() or not 16-byte aligned");

  int dev = 0, sm_count = 0;
  tt_attn_status st = prepare_device(&dev, &sm_count);
  if (st != TT_ATTN_OK) return st;
  if ((st = set_speculative_attributes(dev)) != TT_ATTN_OK) return st;
  const int64_t group = q_heads / kv_heads;
  const TreePlan pl = tree_plan(batch, q_heads, kv_heads, nodes, capacity);
  CUtensorMap tmk, tmv, tmtk, tmtv;
  std::string err;
  if (!encode_map(&tmk, cache_k, cks, &err, tr::KEYS) ||
      !encode_map(&tmv, cache_v, cvs, &err, tr::KEYS) ||
      (pl.persistent && (!encode_map(&tmtk, tree_k, tks, &err, tr::KEYS) ||
                         !encode_map(&tmtv, tree_v, tvs, &err, tr::KEYS))))
    return fail(TT_ATTN_UNSUPPORTED, err);
  tr::Params p{};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_sb = qs.stride[0];
  p.q_sh = qs.stride[1];
  p.q_sn = qs.stride[2];
  p.tk = static_cast<const __nv_bfloat16*>(tree_k);
  p.tk_sb = tks.stride[0];
  p.tk_sh = tks.stride[1];
  p.tk_sn = tks.stride[2];
  p.tv = static_cast<const __nv_bfloat16*>(tree_v);
  p.tv_sb = tvs.stride[0];
  p.tv_sh = tvs.stride[1];
  p.tv_sn = tvs.stride[2];
  p.parents = parents;
  p.parents_sb = parents_stride;
  p.lens = cache_lens;
  p.B = static_cast<int>(batch);
  p.Hkv = static_cast<int>(kv_heads);
  p.G = static_cast<int>(group);
  p.N = static_cast<int>(nodes);
  p.C = static_cast<int>(capacity);
  p.row_tiles = static_cast<int>(pl.row_tiles);
  p.splits = pl.splits;
  p.o = static_cast<__nv_bfloat16*>(out);
  p.lse = lse;
  p.scale_log2 = kScaleLog2;
  if (pl.persistent)
    return launch_tree_persistent(pl, p, workspace, sm_count, tmk, tmv, tmtk, tmtv,
                                  static_cast<cudaStream_t>(stream));
  const Launch launch(dim3(static_cast<unsigned>(batch * kv_heads * pl.row_tiles * pl.splits)),
                      tr::THREADS, tr::kSmemBytes, pl.splits, static_cast<cudaStream_t>(stream));
  const bool multi = pl.row_tiles > 1 || nodes > 16;
  const cudaError_t le =
      multi ? cudaLaunchKernelEx(&launch.cfg, tr::tree_attention_kernel<true>, tmk, tmv, p)
            : cudaLaunchKernelEx(&launch.cfg, tr::tree_attention_kernel<false>, tmk, tmv, p);
  return check_launch("tree_attention_kernel launch", le);
}

TT_ATTN_API tt_attn_status tt_attn_tree_verify_f32(
    const int64_t* tokens, const int32_t* parents, int64_t parents_stride,
    const float* target_probs, int64_t tp_sb, int64_t tp_sn, const float* draft_probs,
    int64_t dp_sb, int64_t dp_sn, const float* uniforms, int64_t batch, int64_t nodes,
    int64_t vocab, int32_t* path, int32_t* counts, int64_t* next_tokens, void* stream) {
  namespace vf = tt::verify;
  if (!tokens || !parents || !target_probs || !uniforms || !path || !counts || !next_tokens)
    return fail(TT_ATTN_BAD_ARG, "tree_verify: tokens, parents, target_probs, uniforms and the "
                                 "outputs must not be NULL");
  if (batch <= 0 || nodes <= 0 || vocab <= 0)
    return fail(TT_ATTN_BAD_ARG, "tree_verify: batch, nodes and vocabulary must be positive");
  if (nodes > TT_ATTN_TREE_MAX_NODES)
    return fail(TT_ATTN_BAD_ARG, "tree_verify: at most 256 nodes per tree");
  if (vocab > TT_ATTN_TREE_MAX_VOCAB)
    return fail(TT_ATTN_BAD_ARG, "tree_verify: at most 4194304 tokens in the vocabulary");
  if (batch > INT32_MAX / vf::MAX_CLUSTER)
    return fail(TT_ATTN_BAD_ARG, "tree_verify: shape exceeds the supported CUDA grid limits");
  if (parents_stride != 0 && parents_stride < nodes)
    return fail(TT_ATTN_BAD_ARG, "tree_verify: parents_stride must be 0 or at least nodes");
  if (tp_sb < 0 || tp_sn < 0 || dp_sb < 0 || dp_sn < 0)
    return fail(TT_ATTN_BAD_ARG, "tree_verify: probability strides must not be negative");
  for (const void* ptr : {static_cast<const void*>(parents), static_cast<const void*>(target_probs),
                          static_cast<const void*>(draft_probs), static_cast<const void*>(uniforms),
                          static_cast<const void*>(path), static_cast<const void*>(counts)})
    if (reinterpret_cast<uintptr_t>(ptr) % 4 != 0)
      return fail(TT_ATTN_BAD_ARG, "tree_verify: pointers must be 4-byte aligned");
  for (const void* ptr : {static_cast<const void*>(tokens), static_cast<const void*>(next_tokens)})
    if (reinterpret_cast<uintptr_t>(ptr) % 8 != 0)
      return fail(TT_ATTN_BAD_ARG, "tree_verify: tokens and next_tokens must be 8-byte aligned");
  int dev = 0;
  tt_attn_status st = prepare_device(&dev);
  if (st != TT_ATTN_OK) return st;
  if ((st = set_speculative_attributes(dev)) != TT_ATTN_OK) return st;
  vf::Params p{};
  p.tokens = tokens;
  p.parents = parents;
  p.parents_sb = parents_stride;
  p.p = target_probs;
  p.p_sb = tp_sb;
  p.p_sn = tp_sn;
  p.q = draft_probs;
  p.q_sb = dp_sb;
  p.q_sn = dp_sn;
  p.u = uniforms;
  p.B = static_cast<int>(batch);
  p.N = static_cast<int>(nodes);
  p.V = static_cast<int>(vocab);
  const int64_t windows = (vocab + vf::WINDOW - 1) / vf::WINDOW;
  // Two CTAs per SM at most, eight windows a CTA at least (4, 8 and 16 measured alike, 32 and 64 up to
  // 7 us slower on 8192 tokens: a warp then takes its windows one after the other).
  p.cluster = static_cast<int>(std::max<int64_t>(
      1, std::min<int64_t>({vf::MAX_CLUSTER, (windows + 7) / 8, 2 * kPlanSms / batch})));
  p.cluster = std::max(
      p.cluster, static_cast<int>((windows + vf::MAX_WINDOWS - 1) / vf::MAX_WINDOWS));
  p.windows = static_cast<int>((windows + p.cluster - 1) / p.cluster);
  const int threads = 32 * std::min(p.windows, vf::MAX_THREADS / 32);
  p.path = path;
  p.counts = counts;
  p.next = next_tokens;
  // 16-byte loads where every row starts on a 16-byte boundary.
  bool vec = vocab % 4 == 0 && tp_sb % 4 == 0 && tp_sn % 4 == 0 && aligned16(target_probs);
  if (draft_probs != nullptr)
    vec = vec && dp_sb % 4 == 0 && dp_sn % 4 == 0 && aligned16(draft_probs);
  const Launch launch(dim3(static_cast<unsigned>(batch * p.cluster)), threads,
                      p.windows * sizeof(unsigned long long), p.cluster,
                      static_cast<cudaStream_t>(stream));
  cudaError_t le;
  if (draft_probs != nullptr)
    le = vec ? cudaLaunchKernelEx(&launch.cfg, vf::tree_verify_kernel<true, true>, p)
             : cudaLaunchKernelEx(&launch.cfg, vf::tree_verify_kernel<true, false>, p);
  else
    le = vec ? cudaLaunchKernelEx(&launch.cfg, vf::tree_verify_kernel<false, true>, p)
             : cudaLaunchKernelEx(&launch.cfg, vf::tree_verify_kernel<false, false>, p);
  return check_launch("tree_verify_kernel launch", le);
}

TT_ATTN_API tt_attn_status tt_attn_tree_commit_bf16(
    void* const* cache_k, const int64_t* ck_strides, void* const* cache_v,
    const int64_t* cv_strides, const void* const* tree_k, const int64_t* tk_strides,
    const void* const* tree_v, const int64_t* tv_strides, int64_t layers, int64_t batch,
    int64_t kv_heads, int64_t nodes, int64_t capacity, int64_t head_dim, const int32_t* path,
    int64_t path_len, const int32_t* counts, const int32_t* cache_lens, int32_t* new_lens,
    void* stream) {
  namespace cm = tt::commit;
  if (!cache_k || !cache_v || !tree_k || !tree_v || !ck_strides || !cv_strides || !tk_strides ||
      !tv_strides || !path || !counts || !cache_lens || !new_lens)
    return fail(TT_ATTN_BAD_ARG, "tree_commit: pointers must not be NULL");
  if (head_dim != TT_ATTN_HEAD_DIM)
    return fail(TT_ATTN_BAD_ARG, "tree_commit currently supports only head_dim=64");
  if (layers <= 0 || batch <= 0 || kv_heads <= 0 || nodes <= 0 || capacity <= 0 || path_len <= 0)
    return fail(TT_ATTN_BAD_ARG, "tree_commit: sizes must be positive");
  if (batch > INT32_MAX / (2 * cm::MAX_LAYERS) || nodes > INT32_MAX || capacity > INT32_MAX ||
      path_len > (INT32_MAX - cm::THREADS) / kv_heads || new_lens == cache_lens)
    return fail(TT_ATTN_BAD_ARG, new_lens == cache_lens
                                     ? "tree_commit: new_lens needs a buffer of its own"
                                     : "tree_commit: shape exceeds the supported CUDA grid limits");
  const Shape4 ck = canonical(batch, kv_heads, capacity, ck_strides);
  const Shape4 cv = canonical(batch, kv_heads, capacity, cv_strides);
  const Shape4 tk = canonical(batch, kv_heads, nodes, tk_strides);
  const Shape4 tv = canonical(batch, kv_heads, nodes, tv_strides);
  for (int64_t l = 0; l < layers; ++l) {
    if (!cache_k[l] || !cache_v[l] || !tree_k[l] || !tree_v[l])
      return fail(TT_ATTN_BAD_ARG, "tree_commit: pointers must not be NULL");
    if (!operand_ok(cache_k[l], ck) || !operand_ok(cache_v[l], cv) || !operand_ok(tree_k[l], tk) ||
        !operand_ok(tree_v[l], tv))
      return fail(TT_ATTN_UNSUPPORTED,
                  "tree_commit: caches and trees need a unit last stride, other strides in "
                  "multiples of 8 elements and 16-byte aligned bases");
  }
  for (const int32_t* ptr : {path, counts, cache_lens, static_cast<const int32_t*>(new_lens)})
    if (reinterpret_cast<uintptr_t>(ptr) % 4 != 0)
      return fail(TT_ATTN_BAD_ARG, "tree_commit: path, counts and lengths must be 4-byte aligned");
  int dev = 0;
  tt_attn_status st = prepare_device(&dev);
  if (st != TT_ATTN_OK) return st;
  for (int64_t first = 0; first < layers; first += cm::MAX_LAYERS) {
    cm::Params p{};
    p.layers = static_cast<int>(std::min<int64_t>(cm::MAX_LAYERS, layers - first));
    for (int l = 0; l < p.layers; ++l) {
      p.cache[0][l] = static_cast<__nv_bfloat16*>(cache_k[first + l]);
      p.cache[1][l] = static_cast<__nv_bfloat16*>(cache_v[first + l]);
      p.tree[0][l] = static_cast<const __nv_bfloat16*>(tree_k[first + l]);
      p.tree[1][l] = static_cast<const __nv_bfloat16*>(tree_v[first + l]);
    }
    p.c_sb[0] = ck.stride[0]; p.c_sh[0] = ck.stride[1]; p.c_st[0] = ck.stride[2];
    p.c_sb[1] = cv.stride[0]; p.c_sh[1] = cv.stride[1]; p.c_st[1] = cv.stride[2];
    p.t_sb[0] = tk.stride[0]; p.t_sh[0] = tk.stride[1]; p.t_st[0] = tk.stride[2];
    p.t_sb[1] = tv.stride[0]; p.t_sh[1] = tv.stride[1]; p.t_st[1] = tv.stride[2];
    p.path = path;
    p.counts = counts;
    p.lens = cache_lens;
    p.new_lens = first == 0 ? new_lens : nullptr;
    p.B = static_cast<int>(batch);
    p.H = static_cast<int>(kv_heads);
    p.N = static_cast<int>(nodes);
    p.C = static_cast<int>(capacity);
    p.P = static_cast<int>(path_len);
    const Launch launch(dim3(static_cast<unsigned>(batch * p.layers * 2)), cm::THREADS, 0, 1,
                        static_cast<cudaStream_t>(stream));
    const cudaError_t le = cudaLaunchKernelEx(&launch.cfg, cm::tree_commit_kernel, p);
    if ((st = check_launch("tree_commit_kernel launch", le)) != TT_ATTN_OK) return st;
  }
  return TT_ATTN_OK;
}

}  // extern "C"
