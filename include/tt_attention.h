/*
 * tt_attention.h - C ABI of the sm_100a (B200) BF16 causal attention forward.
 *
 * Plain C: raw device pointers, element strides and sizes, a CUDA stream passed as
 * `void*` (a cudaStream_t / CUstream), and an integer status. No allocation happens
 * behind these entry points: the caller owns O, LSE and the workspace.
 *
 * Each entry point names the reference interface it replaces (Tiny-transformer,
 * paths relative to that project).
 *
 * Device selection: call with the device that owns the pointers current on the
 * calling thread (cudaSetDevice, or a torch CUDAGuard), as for any CUDA library.
 */
#ifndef TT_ATTENTION_H_
#define TT_ATTENTION_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#define TT_ATTN_API __attribute__((visibility("default")))
#else
#define TT_ATTN_API
#endif

#define TT_ATTN_ABI_VERSION 1
#define TT_ATTN_HEAD_DIM 64

typedef enum tt_attn_status {
  TT_ATTN_OK = 0,
  TT_ATTN_BAD_ARG = 1,     /* invalid sizes, pointers or strides; nothing was launched */
  TT_ATTN_UNSUPPORTED = 2, /* valid request this path cannot take (layout, device);
                              nothing was launched: copy to an aligned contiguous layout */
  TT_ATTN_LAUNCH_FAIL = 3, /* a CUDA call failed; tt_attn_last_error() has the CUDA message */
  TT_ATTN_TIMEOUT = 4      /* a kernel wait ran out (see tt_attn_device_status) */
} tt_attn_status;

/*
 * Causal attention forward, BF16 in / BF16 O / FP32 LSE, head_dim 64.
 *
 * Replaces the BF16 branch of `attention_forward(q, k, v, past_len, segment_ids)`
 * (csrc/attention/attention.cu:32-159, declared in csrc/attention/attention.h:7-9,
 * bound in csrc/attention/bindings.cpp:4-8), i.e. the kernels
 * attention_bf16::forward<EVEN_TILES> (attention_forward_BF16_kernel.cuh:232-389) and
 * decode_partial / decode_merge (attention_decode_BF16_kernel.cuh:45-128).
 *
 *   q        [batch, heads, q_len, 64]  bf16, element strides q_strides[4]
 *   k, v     [batch, heads, kv_len, 64] bf16, element strides k_strides / v_strides
 *            (prefix views of a larger KV cache are read in place)
 *   past_len must equal kv_len - q_len; key j is visible to query row i iff j <= i + past_len.
 *   kv_lens  optional device int32[batch] (q_len must be 1): key j is visible iff
 *            j < kv_lens[b]; values are clamped to [0, kv_len]; 0 gives O = 0, LSE = -inf.
 *   out      contiguous [batch, heads, q_len, 64] bf16
 *   lse      contiguous [batch, heads, q_len] fp32, natural log
 *   workspace / workspace_bytes: device scratch of at least
 *            tt_attn_forward_workspace_size(...) bytes (may be NULL when that is 0). Decode
 *            (q_len == 1) of more than 2^20 (batch * heads * kv_len) K/V rows (2^21 when
 *            batch * heads <= 640) keeps a work
 *            counter and per-sequence arrival counters there, which the call zeroes on
 *            `stream` before its kernel runs, and its split-KV partials; prefill with fewer
 *            256-row query blocks than SMs keeps the partial records of its split blocks.
 *   stream   cudaStream_t the kernels are launched on; no host synchronisation.
 *
 * Layout requirements (else TT_ATTN_UNSUPPORTED): last stride 1, other strides positive
 * multiples of 8 elements, base pointers 16-byte aligned.
 */
TT_ATTN_API tt_attn_status tt_attn_forward_bf16(
    const void* q, const int64_t* q_strides,
    const void* k, const int64_t* k_strides,
    const void* v, const int64_t* v_strides,
    int64_t batch, int64_t heads, int64_t q_len, int64_t kv_len, int64_t head_dim,
    int64_t past_len, const int32_t* kv_lens,
    void* out, float* lse,
    void* workspace, size_t workspace_bytes,
    void* stream);

/* Scratch bytes tt_attn_forward_bf16 needs for this shape: for decode of a cache longer than
 * 1024 keys, a 256-byte work counter, plus (when sequences are split into more than one chunk)
 * one 4-byte arrival counter per (batch, head) rounded up to 256 bytes and 272 bytes of FP32
 * partial per (batch, head, chunk). Replaces the partials tensor the reference allocates
 * (attention.cu:128-129). Returns 0 for decode of caches of up to 1024 keys (one CTA per
 * sequence, no scratch), for prefill shapes and for invalid shapes. */
TT_ATTN_API size_t tt_attn_forward_workspace_size(int64_t batch, int64_t heads, int64_t q_len,
                                                  int64_t kv_len);

/* 1 when a [.., .., .., 64] bf16 operand at `ptr` with these element strides can be read
 * in place; 0 when it must first be copied to aligned contiguous storage.
 * Replaces the alignment decision of aligned_contiguous (attention.cu:20-29). */
TT_ATTN_API int tt_attn_layout_supported(const void* ptr, const int64_t* strides);

/* 1 when the current device can run the kernels (compute capability 10.x), else 0.
 * Replaces the SM80 capability check (attention.cu:72-73). */
TT_ATTN_API int tt_attn_device_supported(void);

/* Reads (and, when clear != 0, resets) the current device's kernel status bits:
 * bit 0 = a bounded wait inside a kernel ran out (returns TT_ATTN_TIMEOUT);
 * bit 1 = tt_rope_append_bf16, tt_attn_cache4_append_bf16, tt_attn_cache4_read_bf16 or
 * tt_attn_qkv_norm_rope_bf16 met a device-held position outside the cache or the table, or
 * tt_attn_tree_commit_bf16 a row or path entry outside its buffer, and skipped those rows
 * (returns TT_ATTN_BAD_ARG). Synchronises the device. */
TT_ATTN_API tt_attn_status tt_attn_device_status(unsigned* flags, int clear);

/*
 * BF16 causal attention backward: dQ, dK, dV from the forward's inputs, output O and LSE.
 *
 * Replaces `attention_backward(q, k, v, dO, O, lse, past_len, segment_ids)`
 * (csrc/attention/attention.cu:161-234, declared in csrc/attention/attention.h, bound in
 * csrc/attention/bindings.cpp), i.e. the preprocess, dKdV and dQ kernels
 * (attention_backward_preprocess_kernel.cuh, attention_backward_dKdV_kernel.cu,
 * attention_backward_dQ_kernel.cu). Same arithmetic: D = rowsum(dO * O), P = exp(S / 8 - LSE),
 * dS = P * (dO.V^T - D), P and dS rounded to bf16 before the products, FP32 accumulation,
 * dQ = dS.K / 8, dK = dS^T.Q / 8, dV = P^T.dO.
 *
 *   q, k, v     [batch, heads, q_len | kv_len, 64] bf16 with element strides (same layout rules
 *               as tt_attn_forward_bf16; TT_ATTN_UNSUPPORTED otherwise)
 *   dout, out   contiguous [batch, heads, q_len, 64] bf16 (dO and the forward's O)
 *   lse         contiguous [batch, heads, q_len] FP32, natural log (the forward's LSE)
 *   dq          contiguous [batch, heads, q_len, 64] bf16 output
 *   dk, dv      contiguous [batch, heads, kv_len, 64] bf16 outputs
 *   workspace   tt_attn_backward_workspace_size() bytes, 16-byte aligned (the FP32 row sums D,
 *               the FP32 dQ accumulator and a work counter; its contents on entry do not matter)
 *
 * Mask: key j visible to query i iff j <= i + past_len, kv_len == q_len + past_len.
 * On `stream`, in order, three kernels: row sums D (which also zeroes the dQ accumulator and
 * the work counter), one persistent dQ/dK/dV kernel, dQ scaling to bf16. Nothing is allocated.
 */
TT_ATTN_API tt_attn_status tt_attn_backward_bf16(
    const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
    const void* v, const int64_t* v_strides, const void* dout, const void* out, const float* lse,
    int64_t batch, int64_t heads, int64_t q_len, int64_t kv_len, int64_t head_dim,
    int64_t past_len, void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes,
    void* stream);

/*
 * Same contract as tt_attn_backward_bf16, with bit-identical results on every call: each output
 * element is accumulated by one CTA in a fixed order (three kernels: row sums D, a dQ kernel
 * over 128-row query tiles, a dK/dV kernel over 128-key tiles), where tt_attn_backward_bf16
 * adds the dQ contributions of different key tiles with reduce-adds in timing-dependent order.
 * The torch binding takes this path under torch.use_deterministic_algorithms(True); the
 * reference's own backward kernels use no atomics. Same workspace size.
 */
TT_ATTN_API tt_attn_status tt_attn_backward_bf16_deterministic(
    const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
    const void* v, const int64_t* v_strides, const void* dout, const void* out, const float* lse,
    int64_t batch, int64_t heads, int64_t q_len, int64_t kv_len, int64_t head_dim,
    int64_t past_len, void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes,
    void* stream);

/* Bytes of workspace tt_attn_backward_bf16 needs (batch * heads * q_len FP32 row sums, padded
 * to 256 bytes, plus batch * heads * q_len * 64 FP32 for dQ), 0 for invalid sizes. */
TT_ATTN_API size_t tt_attn_backward_workspace_size(int64_t batch, int64_t heads, int64_t q_len);

/*
 * Fused rotary embedding + KV-cache append for one decoder layer (the step before attention
 * in Block.forward, tiny_transformer/model.py:61-68: reference.rope on q and k, reference.py:
 * 30-34, then KVCache.update, model.py:29-41). Replaces for this path the reference's
 * `rope` operator calls (student rope_forward) plus the two cache copies.
 *
 *   qkv      [batch, q_len, 3, heads, 64] bf16, contiguous (the fused QKV projection)
 *   cos, sin [table_len, 32] FP32 contiguous, row = position (rounded to bf16 as the
 *            reference's cos.to(x.dtype) does)
 *   q_out    [batch, heads, q_len, 64] bf16 contiguous: rope(q)
 *   cache_k / cache_v [batch, heads, capacity, 64] bf16, last stride 1, element strides in
 *            ck_strides / cv_strides (4 entries); row `position + t` receives rope(k) / v.
 *
 * The start position is `position` or, when `position_dev` is not NULL, the int64 it points
 * to on the device (read at run time, so a captured CUDA graph can serve every step). Host
 * positions are validated here (BAD_ARG); device-held ones by the kernel, which skips rows
 * outside [0, min(capacity, table_len)) and sets status bit 1. Bit-exact with the reference's
 * bf16 expression. All pointers 4-byte aligned; 16-byte aligned rows are fastest.
 */
TT_ATTN_API tt_attn_status tt_rope_append_bf16(
    const void* qkv, int64_t batch, int64_t q_len, int64_t heads, const float* cos,
    const float* sin, int64_t table_len, int64_t position, const int64_t* position_dev,
    void* q_out, void* cache_k, const int64_t* ck_strides, void* cache_v,
    const int64_t* cv_strides, int64_t capacity, void* stream);

/* QKV projection with RoPE and the KV-cache append in its epilogue, one kernel per layer: the
 * steps in front of the attention in the reference's Block.forward (model.py:59-67:
 * `linear(normalized, qkv)`, `rope(q)`, `rope(k)`, `KVCache.update`), with the projection never
 * written to memory.
 *   hidden   [batch * q_len, dim] bf16 row-major (the normalised hidden state), dim % 64 == 0
 *   w_qkv    [3 * heads * 64, dim] bf16 row-major (the layer's qkv weight)
 *   cos/sin  [table_len, 32] FP32 tables; position: first position (or position_dev, an int64
 *            on the device read at run time)
 *   q_out    [batch, heads, q_len, 64] bf16 contiguous = rope(q)
 *   cache_k/cache_v [batch, heads, capacity, 64] bf16 (unit last stride): rows position + t get
 *            rope(k) and v.
 * The projection is accumulated in FP32 and rounded to bf16, then rotated exactly as
 * tt_rope_append_bf16 rotates a bf16 projection. All pointers 16-byte aligned. The feature
 * tile width (16 to 128 features) is chosen per call so that the grid covers the SMs; the
 * result does not depend on it. */
TT_ATTN_API tt_attn_status tt_qkv_rope_append_bf16(
    const void* hidden, int64_t batch, int64_t q_len, int64_t dim, const void* w_qkv,
    int64_t heads, const float* cos, const float* sin, int64_t table_len, int64_t position,
    const int64_t* position_dev, void* q_out, void* cache_k, const int64_t* ck_strides,
    void* cache_v, const int64_t* cv_strides, int64_t capacity, void* stream);

/* Diagnostic for the failure path: launches one warp on `stream` that waits on a barrier
 * phase nothing completes, bounded by `budget_cycles` (1 .. 1e9 SM clock cycles). The wait
 * gives up by itself and sets bit 0 of the device status, which the caller then reads (and
 * clears) with tt_attn_device_status; the context stays usable. No counterpart in the
 * reference, which has no bounded waits. Returns BAD_ARG for a budget outside the range. */
TT_ATTN_API tt_attn_status tt_attn_selftest_wait_timeout(int64_t budget_cycles, void* stream);

/* Human-readable name of a status code. */
TT_ATTN_API const char* tt_attn_status_string(tt_attn_status status);

/* Message for the last non-OK status returned on the calling thread ("" if none). */
TT_ATTN_API const char* tt_attn_last_error(void);

TT_ATTN_API int tt_attn_abi_version(void);

/*
 * Single-token decode that allocates nothing, not even through the caller. No counterpart in
 * the reference: it exists for callers that cannot allocate device memory when they decode
 * (a server whose memory is entirely reserved by its own pools, a Go/Java/Rust host calling
 * this C ABI without a CUDA allocator, a loop that must stay out of the driver's allocator).
 *
 * Same computation and arguments as tt_attn_forward_bf16 with q_len = 1, head_dim = 64 and
 * past_len = kv_len - 1; the split-KV partials live in a static device array of 8 MiB
 * (8388608 bytes) that every GPU loading this library holds until exit. Shapes whose partials
 * exceed it (tt_attn_forward_workspace_size) return TT_ATTN_BAD_ARG; a device other than
 * sm_100 returns TT_ATTN_UNSUPPORTED. The first call on a device looks up the array's device
 * address (with that device current), and so does the first call after the current context
 * of that device changed (cudaDeviceReset, or a context the caller made current); make those
 * calls before any stream capture. All calls share the array: calls whose kernels overlap on
 * the GPU (different streams, or different host threads) race on it and must be serialised
 * by the caller. Caches of up to 2^20 (batch * heads * kv_len) K/V rows, or up to 2^21 in at
 * most 640 (batch, head) sequences, use no scratch at all.
 */
TT_ATTN_API tt_attn_status tt_attn_decode_bf16_noalloc(
    const void* q, const int64_t* q_strides,
    const void* k, const int64_t* k_strides,
    const void* v, const int64_t* v_strides,
    int64_t batch, int64_t heads, int64_t kv_len, const int32_t* kv_lens,
    void* out, float* lse, void* stream);

/* ------------------------------------------------------------------ speculative decoding
 * Three operators around one step of speculative decoding. A draft proposes a tree of `nodes`
 * tokens per sequence; the target runs once over all of them (attention by
 * tt_attn_tree_forward_bf16, each node seeing the cached prefix and its own branch), the walk
 * through the tree is decided by tt_attn_tree_verify_f32, and the accepted path's K/V rows are
 * appended to the caches by tt_attn_tree_commit_bf16. The drafted tokens' K/V rows stay outside
 * the cache until then. No counterpart in the reference, which generates one token at a time
 * (tiny_transformer/generate.py).
 *
 * A tree is given by `parents`: int32 device [nodes] (parents_stride 0, one tree for the batch)
 * or [batch, nodes] rows parents_stride elements apart. parents[n] is a lower index, or -1 for a
 * root. A node whose chain of parents does not reach -1 over strictly lower indices is not in use
 * (padding of a smaller tree): nobody sees it, and its own output is empty.
 */
#define TT_ATTN_TREE_MAX_NODES 256
#define TT_ATTN_TREE_MAX_VOCAB 4194304

/*
 * Attention of the tree's nodes: node n of sequence b attends to cache rows [0, cache_lens[b]) and
 * to the tree rows of its chain (itself, its parent, ... up to the root). Scale 1/8, FP32 softmax.
 *
 *   q          [batch, q_heads, nodes, 64] bf16; q_heads a multiple of kv_heads: query head h
 *              reads K/V head h / (q_heads / kv_heads)
 *   tree_k/v   [batch, kv_heads, nodes, 64] bf16, the drafted tokens' own rows
 *   cache_k/v  [batch, kv_heads, capacity, 64] bf16
 *   cache_lens optional device int32[batch], clamped to [0, capacity]; NULL: the whole capacity
 *   out        contiguous [batch, q_heads, nodes, 64] bf16, 16-byte aligned
 *   lse        optional contiguous [batch, q_heads, nodes] fp32, natural log
 *   workspace  tt_attn_tree_workspace_size() bytes, 16-byte aligned (may be NULL when that is 0)
 *
 * Nodes not in use get O = 0, LSE = -inf. What a node does not see does not change its output,
 * whatever it holds (NaN and infinities included); an infinity in a cached V row that is seen makes
 * that feature of the output infinite or NaN. 1 <= nodes <= TT_ATTN_TREE_MAX_NODES. Layout
 * rules of q and all K/V tensors as for tt_attn_forward_bf16 (TT_ATTN_UNSUPPORTED otherwise).
 */
TT_ATTN_API tt_attn_status tt_attn_tree_forward_bf16(
    const void* q, const int64_t* q_strides, const void* tree_k, const int64_t* tk_strides,
    const void* tree_v, const int64_t* tv_strides, const void* cache_k, const int64_t* ck_strides,
    const void* cache_v, const int64_t* cv_strides, int64_t batch, int64_t q_heads,
    int64_t kv_heads, int64_t nodes, int64_t capacity, int64_t head_dim, const int32_t* parents,
    int64_t parents_stride, const int32_t* cache_lens, void* out, float* lse, void* workspace,
    size_t workspace_bytes, void* stream);

/* Scratch bytes tt_attn_tree_forward_bf16 needs for this shape; 0 for invalid shapes too. */
TT_ATTN_API size_t tt_attn_tree_workspace_size(int64_t batch, int64_t q_heads, int64_t kv_heads,
                                               int64_t nodes, int64_t capacity);

/*
 * Walk of the tree with given random numbers (speculative sampling). From node 0 the children of
 * the current node are tried in index order: a child with token t is accepted with probability
 * min(1, p(t) / q(t)), otherwise p becomes max(p - q, 0), renormalised, for the next child; when
 * no child is accepted, the next token is drawn from what is left of p.
 *
 *   tokens        int64 device [batch, nodes] contiguous: token of each node (node 0's is not read
 *                 as a candidate). A token outside [0, vocab) is never accepted.
 *   target_probs  fp32 device [batch, nodes, vocab], unit last stride, element strides tp_sb, tp_sn:
 *                 row n is the target's distribution of the token after node n
 *   draft_probs   fp32 likewise (dp_sb, dp_sn): the distribution that n's children were drawn from.
 *                 NULL: children were chosen, not drawn (q = 1 at the child's token)
 *   uniforms      fp32 device [batch, nodes] contiguous in [0, 1): entry n decides node n, entry 0
 *                 draws the next token
 *   path          int32 [batch, nodes]: the accepted nodes from the root (node 0) on, then -1
 *   counts        int32 [batch]: accepted nodes, the root included (0 when node 0 is not a root)
 *   next_tokens   int64 [batch]: the token after the path (-1 where counts is 0, or where no token
 *                 has any weight)
 *
 * Weights are whole numbers (probabilities times 2^36, rounded down), so results do not depend on
 * the order of any sum; the exact definition is at the kernel. Uniforms that are 2^-24 apart, as FP32
 * generators draw them, resolve the next token's probabilities to 2^-24. Probabilities are taken into
 * [0, 1], NaN as 0. 1 <= nodes <= TT_ATTN_TREE_MAX_NODES, vocab <= TT_ATTN_TREE_MAX_VOCAB.
 */
TT_ATTN_API tt_attn_status tt_attn_tree_verify_f32(
    const int64_t* tokens, const int32_t* parents, int64_t parents_stride,
    const float* target_probs, int64_t tp_sb, int64_t tp_sn, const float* draft_probs,
    int64_t dp_sb, int64_t dp_sn, const float* uniforms, int64_t batch, int64_t nodes,
    int64_t vocab, int32_t* path, int32_t* counts, int64_t* next_tokens, void* stream);

/*
 * Append of the accepted path to the caches of `layers` layers: row i < counts[b] of sequence b
 * goes from tree row path[b, i] to cache row cache_lens[b] + i, keys and values, all layers.
 *
 *   cache_k/v, tree_k/v  host arrays of `layers` device pointers; every layer has the same shape and
 *                        strides: caches [batch, kv_heads, capacity, 64], trees [batch, kv_heads,
 *                        nodes, 64] bf16, last stride 1, other strides multiples of 8, 16-byte
 *                        aligned bases (TT_ATTN_UNSUPPORTED otherwise)
 *   path                 int32 device [batch, path_len] contiguous
 *   counts, cache_lens   int32 device [batch]
 *   new_lens             int32 device [batch]: cache_lens[b] + the rows that fit. A buffer
 *                        of its own: the kernel's blocks read cache_lens while it is written
 *
 * Rows that do not fit the capacity and path entries outside [0, nodes) are skipped and set bit 1
 * of the device status (tt_attn_device_status). The row of such a path entry is not written but
 * counts in new_lens, as later rows of the path keep their places: after that status the rows
 * appended to the sequence must not be used. The caches must not overlap the trees.
 */
TT_ATTN_API tt_attn_status tt_attn_tree_commit_bf16(
    void* const* cache_k, const int64_t* ck_strides, void* const* cache_v,
    const int64_t* cv_strides, const void* const* tree_k, const int64_t* tk_strides,
    const void* const* tree_v, const int64_t* tv_strides, int64_t layers, int64_t batch,
    int64_t kv_heads, int64_t nodes, int64_t capacity, int64_t head_dim, const int32_t* path,
    int64_t path_len, const int32_t* counts, const int32_t* cache_lens, int32_t* new_lens,
    void* stream);

/* ------------------------------------------------------------------ query/key norm
 * RMS norm of every query and key head of a fused QKV projection with the rotary embedding in the same
 * pass. No counterpart in the reference, whose blocks norm the hidden state only (tiny_transformer/model.py:46-76)
 * and rotate in operations of their own (reference.py:30-34).
 *
 *   qkv        [batch, q_len, q_heads + 2 kv_heads, 64] bf16 (query, key, value heads), features adjacent, element
 *              strides qkv_strides[3] (batch, token, head) in multiples of 8, 16-byte aligned
 *              (TT_ATTN_UNSUPPORTED otherwise)
 *   q_weight, k_weight  [64] bf16, or FP32 with weights_f32 != 0, 16-byte aligned; both NULL: no norm, the
 *              rotation alone
 *   cos, sin   [table_len, 32] FP32, row = position, 16-byte aligned; used in FP32
 *   position   of token 0 (validated here), or position_dev: token (b, t) is at
 *              position_dev[b * position_sb + t * position_st], + t where position_st is 0
 *   q_out      contiguous [batch, q_heads, q_len, 64] bf16; k_out [batch, kv_heads, q_len, 64]
 *
 * For a head x of weight w: n = x w / sqrt(mean(x^2) + eps), then adjacent pairs (n_2i, n_2i+1) are turned by the
 * table row of the position. FP32, rounded to bf16 once. Rows whose device-held position is outside the table are
 * zero and set status bit 1.
 */
TT_ATTN_API tt_attn_status tt_attn_qkv_norm_rope_bf16(
    const void* qkv, const int64_t* qkv_strides, int64_t batch, int64_t q_len, int64_t q_heads,
    int64_t kv_heads, const void* q_weight, const void* k_weight, int weights_f32, const float* cos,
    const float* sin, int64_t table_len, int64_t position, const int64_t* position_dev,
    int64_t position_sb, int64_t position_st, double eps, void* q_out, void* k_out, void* stream);

/*
 * Gradients of tt_attn_qkv_norm_rope_bf16: its arguments, then
 *   dq, dk, dv   [batch, heads, q_len, 64] bf16 with element strides (layout rules of tt_attn_forward_bf16): the
 *                gradients of q_out, k_out and of the value heads; NULL: zero
 *   dqkv         contiguous [batch, q_len, q_heads + 2 kv_heads, 64] bf16, dv copied into its value heads
 *   dq_weight, dk_weight  [64] in the weights' type (not used without weights)
 *   workspace    tt_attn_qkv_norm_rope_backward_workspace_size() bytes, 16-byte aligned (not used without weights)
 * The weights' gradients are added in a fixed order: the same inputs give the same bits.
 */
TT_ATTN_API tt_attn_status tt_attn_qkv_norm_rope_backward_bf16(
    const void* qkv, const int64_t* qkv_strides, int64_t batch, int64_t q_len, int64_t q_heads,
    int64_t kv_heads, const void* q_weight, const void* k_weight, int weights_f32, const float* cos,
    const float* sin, int64_t table_len, int64_t position, const int64_t* position_dev,
    int64_t position_sb, int64_t position_st, double eps, const void* dq, const int64_t* dq_strides,
    const void* dk, const int64_t* dk_strides, const void* dv, const int64_t* dv_strides, void* dqkv,
    void* dq_weight, void* dk_weight, void* workspace, size_t workspace_bytes, void* stream);

TT_ATTN_API size_t tt_attn_qkv_norm_rope_backward_workspace_size(void);

/* ------------------------------------------------------------------ 4-bit KV cache
 * A KV cache of 36 bytes a row (128 in bf16): rows are quantised as they are written, read back as bf16, and
 * attended to without ever being expanded in memory. No counterpart in the reference, whose cache has the model's
 * type (tiny_transformer/model.py:11-43).
 *
 * A cache is [batch, kv_heads, blocks, 576] bytes, byte strides c*_strides[4] (last 1, others multiples of 16, at least
 * 576), 16-byte aligned (TT_ATTN_UNSUPPORTED otherwise); its capacity is 16 * blocks rows. A block holds 16 rows:
 *   bytes 0-511    codes, row r at 32 r: feature 2i in the low half of byte i, 2i + 1 in the high half; a code is e2m1
 *                  (bit 3 the sign, then 0 0.5 1 1.5 2 3 4 6)
 *   bytes 512-575  scales, row r at 512 + 4 r, one for 16 features: the upper byte of a half without its sign (5
 *                  bits of exponent, 3 of mantissa), at most 0xE2 = 10240, or 0xFF = NaN
 * A value is code x scale. 16 values are quantised with scale = max|x| / 6 rounded to nearest even (at most
 * 10240), codes rounded to nearest, ties to the even code, saturating. A group with a NaN gets the scale NaN. Scales have 4
 * significant bits from 2^-14 (max|x| 3.7e-4) to 10240 and fewer down to 2^-17; smaller groups become zero.
 */
#define TT_ATTN_CACHE4_BLOCK_ROWS 16
#define TT_ATTN_CACHE4_BLOCK_BYTES 576
#define TT_ATTN_CACHE4_MAX_QUERIES 16

/*
 * tt_attn_qkv_norm_rope_bf16's pass with the cache append in it: q goes to q_out, the keys (as bf16, rounded from FP64
 * by way of FP32) and the values are quantised into rows position + t of the caches. Other rows are left as they are.
 * position_dev[b * position_sb] + t with a device-held position. Rows outside the cache or the table are not
 * written, their q is zero, and status bit 1 is set.
 * No two blocks may overlap: sorted by stride, each dimension of a cache has to reach past those inside it
 * (TT_ATTN_UNSUPPORTED otherwise), and the two caches must not overlap (TT_ATTN_BAD_ARG); with equal strides one may lie
 * in the other's gaps, as the two halves of [batch, 2, kv_heads, blocks, 576] do.
 */
TT_ATTN_API tt_attn_status tt_attn_cache4_append_bf16(
    const void* qkv, const int64_t* qkv_strides, int64_t batch, int64_t q_len, int64_t q_heads,
    int64_t kv_heads, const void* q_weight, const void* k_weight, int weights_f32, const float* cos,
    const float* sin, int64_t table_len, int64_t position, const int64_t* position_dev,
    int64_t position_sb, double eps, void* q_out, void* cache_k, const int64_t* ck_strides,
    void* cache_v, const int64_t* cv_strides, int64_t blocks, void* stream);

/*
 * Rows start + i, i < rows, of both caches as bf16 (exact): k_out and v_out contiguous [batch, kv_heads, rows, 64].
 * start is validated here; with start_dev, sequence b starts at start_dev[b * start_sb], and rows outside the
 * cache read as zero and set status bit 1.
 */
TT_ATTN_API tt_attn_status tt_attn_cache4_read_bf16(
    const void* cache_k, const int64_t* ck_strides, const void* cache_v, const int64_t* cv_strides,
    int64_t batch, int64_t kv_heads, int64_t blocks, int64_t start, const int64_t* start_dev,
    int64_t start_sb, int64_t rows, void* k_out, void* v_out, void* stream);

/*
 * Attention of the last q_len tokens of each sequence, whose rows are in the caches: query t of sequence b sees
 * rows j < kv_lens[b] - (q_len - 1 - t). Scale 1/8, FP32 softmax.
 *
 *   q         [batch, q_heads, q_len, 64] bf16 (layout rules of tt_attn_forward_bf16), 1 <= q_len <=
 *             TT_ATTN_CACHE4_MAX_QUERIES; q_heads a multiple of kv_heads: query head h reads K/V head
 *             h / (q_heads / kv_heads)
 *   kv_lens   optional device int32[batch], clamped to [0, 16 * blocks]; NULL: the whole capacity
 *   out       contiguous [batch, q_heads, q_len, 64] bf16, 16-byte aligned
 *   lse       optional contiguous [batch, q_heads, q_len] FP32, natural log
 *   workspace tt_attn_cache4_workspace_size() bytes, 16-byte aligned (may be NULL when that is 0)
 *
 * A query that sees no row gets O = 0, LSE = -inf. Rows that a query does not see never change its output, whatever
 * they hold.
 */
TT_ATTN_API tt_attn_status tt_attn_cache4_forward_bf16(
    const void* q, const int64_t* q_strides, const void* cache_k, const int64_t* ck_strides,
    const void* cache_v, const int64_t* cv_strides, int64_t batch, int64_t q_heads, int64_t kv_heads,
    int64_t q_len, int64_t blocks, int64_t head_dim, const int32_t* kv_lens, void* out, float* lse,
    void* workspace, size_t workspace_bytes, void* stream);

/* Scratch bytes tt_attn_cache4_forward_bf16 needs for this shape; 0 for invalid shapes too. */
TT_ATTN_API size_t tt_attn_cache4_workspace_size(int64_t batch, int64_t q_heads, int64_t kv_heads,
                                                 int64_t q_len, int64_t blocks);

#ifdef __cplusplus
}
#endif

#endif /* TT_ATTENTION_H_ */
