// PyTorch extension `tt_attention_C`: the reference's native operator surface
// (`attention_forward(q, k, v, past_len=0, segment_ids=None) -> (O, LSE)`, Tiny-transformer
// csrc/attention/bindings.cpp:4-8, attention.cu:32-159) on top of the C ABI in
// include/tt_attention.h. This file owns validation (same checks and message fragments as
// csrc/attention/attention_common.h:9-87 and attention.cu:36-73), output / workspace
// allocation through the caching allocator, and the layout decision; all device work goes
// through tt_attn_forward_bf16 on the current stream.
#include <torch/extension.h>

#include <ATen/autocast_mode.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cstdint>
#include <limits>
#include <optional>
#include <tuple>
#include <vector>

#include "tt_attention.h"

namespace {

void check_tensors(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v) {
  for (const auto* t : {&q, &k, &v}) {
    TORCH_CHECK(t->defined(), "attention inputs must be defined");
    TORCH_CHECK(t->is_cuda(), "All inputs must be CUDA tensors");
  }
  for (const auto* t : {&q, &k, &v}) {
    TORCH_CHECK(t->device() == q.device(), "All inputs must be on the same device");
    TORCH_CHECK(t->scalar_type() == at::kFloat || t->scalar_type() == at::kBFloat16,
                "attention supports only float32 and bf16 inputs");
    TORCH_CHECK(t->scalar_type() == q.scalar_type(), "q, k, v must have the same dtype");
    TORCH_CHECK(t->layout() == at::kStrided, "All inputs must be strided tensors");
  }
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, "q, k, v must be a 4D tensor");
  TORCH_CHECK(k.size(0) == q.size(0) && v.size(0) == q.size(0),
              "q, k, v must have the same first dimension");
  TORCH_CHECK(k.size(1) == q.size(1) && v.size(1) == q.size(1),
              "q, k, v must have the same second dimension");
  TORCH_CHECK(k.size(3) == q.size(3) && v.size(3) == q.size(3),
              "q, k, v must have the same last dimension");
  TORCH_CHECK(q.size(3) == TT_ATTN_HEAD_DIM, "attention currently supports only head_dim=64");
  TORCH_CHECK(q.size(0) > 0 && q.size(1) > 0 && q.size(2) > 0 && k.size(2) > 0,
              "attention batch, heads and sequence lengths must be positive");
}

void check_mask(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v,
                int64_t past_len) {
  TORCH_CHECK(past_len >= 0, "past_len must be non-negative");
  TORCH_CHECK(v.size(2) == k.size(2), "k and v must have the same sequence length");
  // Subtract instead of adding: past_len + Tq may overflow.
  TORCH_CHECK(k.size(2) >= q.size(2) && past_len == k.size(2) - q.size(2),
              "expected Tk == past_len + Tq");
}

bool readable_in_place(const torch::Tensor& x) {
  const int64_t st[4] = {x.stride(0), x.stride(1), x.stride(2), x.stride(3)};
  int64_t canon[4] = {st[0], st[1], st[2], st[3]};
  // Size-1 dimensions are never stepped over; their stride does not matter.
  const int64_t contiguous[3] = {x.size(1) * x.size(2) * x.size(3), x.size(2) * x.size(3),
                                 x.size(3)};
  for (int d = 0; d < 3; ++d)
    if (x.size(d) == 1) canon[d] = contiguous[d];
  return tt_attn_layout_supported(x.data_ptr(), canon) != 0;
}

// Same fallback as the reference's aligned_contiguous (attention.cu:20-29), taken only
// when the TMA / bulk-copy path cannot read the view in place.
torch::Tensor aligned_contiguous(torch::Tensor x) {
  if (readable_in_place(x)) return x;
  x = x.contiguous();
  if (reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 != 0) x = x.clone();
  return x;
}

}  // namespace

std::tuple<torch::Tensor, torch::Tensor> attention_forward(
    torch::Tensor q, torch::Tensor k, torch::Tensor v, int64_t past_len,
    std::optional<torch::Tensor> segment_ids, std::optional<torch::Tensor> kv_lens) {
  check_tensors(q, k, v);
  check_mask(q, k, v, past_len);
  TORCH_CHECK(!(at::GradMode::is_enabled() &&
                (q.requires_grad() || k.requires_grad() || v.requires_grad())),
              "student attention backward requires the Python autograd binding; "
              "use student.attention or no_grad for inference");
  TORCH_CHECK(q.scalar_type() == at::kBFloat16,
              "float32 attention is not provided by the sm_100a path; pass bf16 q, k, v");
  TORCH_CHECK(!segment_ids.has_value(), "segment_ids is not supported for bf16 kernel");
  const int64_t B = q.size(0), H = q.size(1), Tq = q.size(2), Tk = k.size(2);
  const int64_t max_grid = std::numeric_limits<int32_t>::max();
  const int64_t q_tiles = (Tq + 127) / 128;
  // Divide before multiplying: B * H * tiles must fit grid.x.
  TORCH_CHECK(q_tiles <= max_grid && B <= max_grid / q_tiles / H,
              "attention shape exceeds the supported CUDA grid limits");
  TORCH_CHECK(Tk <= std::numeric_limits<int32_t>::max(),
              "bf16 attention sequence lengths must fit int32 (Tk <= INT32_MAX)");
  if (kv_lens.has_value()) {
    const auto& lens = *kv_lens;
    TORCH_CHECK(lens.defined() && lens.is_cuda() && lens.device() == q.device(),
                "kv_lens must be a CUDA tensor on the same device as q");
    TORCH_CHECK(lens.scalar_type() == at::kInt || lens.scalar_type() == at::kLong,
                "kv_lens must be int32 or int64");
    TORCH_CHECK(lens.dim() == 1 && lens.size(0) == B, "kv_lens must have shape [B]");
    TORCH_CHECK(Tq == 1, "kv_lens requires single-token decode (Tq == 1)");
  }

  const c10::cuda::CUDAGuard device_guard(q.device());
  const auto* props = at::cuda::getDeviceProperties(q.get_device());
  TORCH_CHECK(props->major == 10,
              "the bf16 attention kernels require an sm_100 GPU (compute capability 10.x); "
              "found SM", props->major, props->minor);
  auto stream = c10::cuda::getCurrentCUDAStream(q.get_device());

  q = aligned_contiguous(q);
  k = aligned_contiguous(k);
  v = aligned_contiguous(v);
  torch::Tensor lens32;
  if (kv_lens.has_value()) lens32 = kv_lens->to(at::kInt).contiguous();

  auto o = torch::empty({B, H, Tq, TT_ATTN_HEAD_DIM}, q.options());
  auto lse = torch::empty({B, H, Tq}, q.options().dtype(at::kFloat));
  const size_t ws_bytes = tt_attn_forward_workspace_size(B, H, Tq, Tk);
  torch::Tensor ws;
  if (ws_bytes > 0)
    ws = torch::empty({static_cast<int64_t>(ws_bytes)}, q.options().dtype(at::kByte));

  const int64_t qs[4] = {q.stride(0), q.stride(1), q.stride(2), q.stride(3)};
  const int64_t ks[4] = {k.stride(0), k.stride(1), k.stride(2), k.stride(3)};
  const int64_t vs[4] = {v.stride(0), v.stride(1), v.stride(2), v.stride(3)};
  const tt_attn_status st = tt_attn_forward_bf16(
      q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, B, H, Tq, Tk, TT_ATTN_HEAD_DIM,
      past_len, lens32.defined() ? lens32.data_ptr<int32_t>() : nullptr, o.data_ptr(),
      lse.data_ptr<float>(), ws_bytes > 0 ? ws.data_ptr() : nullptr, ws_bytes,
      static_cast<void*>(stream.stream()));
  TORCH_CHECK(st == TT_ATTN_OK, "tt_attn_forward_bf16 failed: ", tt_attn_status_string(st),
              ": ", tt_attn_last_error());
  return {o, lse};
}

void check_upstream(const torch::Tensor& q, const torch::Tensor& dO, const torch::Tensor& o,
                    const torch::Tensor& lse) {
  for (const torch::Tensor* x : {&dO, &o, &lse}) {
    TORCH_CHECK(x->defined(), "dO, O and LSE must be defined");
    TORCH_CHECK(x->is_cuda() && x->device() == q.device(),
                "dO, O and LSE must be CUDA tensors on the same device as q");
    TORCH_CHECK(x->layout() == at::kStrided, "dO, O and LSE must have strided layout");
  }
  TORCH_CHECK(dO.scalar_type() == q.scalar_type() && o.scalar_type() == q.scalar_type(),
              "dO and O must have the same dtype as q");
  TORCH_CHECK(dO.sizes() == q.sizes() && o.sizes() == q.sizes(),
              "dO and O must have the same shape as q");
  TORCH_CHECK(lse.scalar_type() == at::kFloat, "LSE must be float32");
  TORCH_CHECK(lse.dim() == 3 && lse.size(0) == q.size(0) && lse.size(1) == q.size(1) &&
                  lse.size(2) == q.size(2),
              "LSE must have shape [B, Nh, Tq]");
}

// Contiguous, 16-byte aligned copy of x unless it already is one.
torch::Tensor contiguous_aligned(torch::Tensor x) {
  x = x.contiguous();
  if (reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 != 0) x = x.clone();
  return x;
}

// The reference's native backward (attention.cu:161-234): same argument order, validation
// order and message fragments; all device work through tt_attn_backward_bf16.
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> attention_backward(
    torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor dO, torch::Tensor O,
    torch::Tensor lse, int64_t past_len, std::optional<torch::Tensor> segment_ids) {
  check_tensors(q, k, v);
  check_mask(q, k, v, past_len);
  TORCH_CHECK(q.scalar_type() == at::kBFloat16, "student attention backward supports only bf16");
  TORCH_CHECK(!segment_ids.has_value(),
              "segment_ids is not supported for bf16 attention backward");
  check_upstream(q, dO, O, lse);
  const int64_t B = q.size(0), H = q.size(1), Tq = q.size(2), Tk = k.size(2);
  TORCH_CHECK(Tk <= std::numeric_limits<int32_t>::max(),
              "bf16 attention sequence lengths must fit int32 (Tk <= INT32_MAX)");
  const int64_t max_grid = std::numeric_limits<int32_t>::max();
  const int64_t k_tiles = (Tk + 127) / 128;  // >= query tiles
  TORCH_CHECK(B <= max_grid / H && k_tiles <= max_grid / (B * H),
              "attention backward shape exceeds the supported CUDA grid limits");
  const c10::cuda::CUDAGuard device_guard(q.device());
  const auto* props = at::cuda::getDeviceProperties(q.get_device());
  TORCH_CHECK(props->major == 10,
              "the bf16 attention kernels require an sm_100 GPU (compute capability 10.x); "
              "found SM", props->major, props->minor);
  auto stream = c10::cuda::getCurrentCUDAStream(q.get_device());
  // Validated; now materialise the layouts the kernels read (on the current stream).
  q = aligned_contiguous(q);
  k = aligned_contiguous(k);
  v = aligned_contiguous(v);
  dO = contiguous_aligned(dO);
  O = contiguous_aligned(O);
  lse = lse.contiguous();
  auto dq = torch::empty({B, H, Tq, TT_ATTN_HEAD_DIM}, q.options());
  auto dk = torch::empty({B, H, Tk, TT_ATTN_HEAD_DIM}, q.options());
  auto dv = torch::empty({B, H, Tk, TT_ATTN_HEAD_DIM}, q.options());
  const size_t ws_bytes = tt_attn_backward_workspace_size(B, H, Tq);
  auto ws = torch::empty({static_cast<int64_t>(ws_bytes)}, q.options().dtype(at::kByte));
  const int64_t qs[4] = {q.stride(0), q.stride(1), q.stride(2), q.stride(3)};
  const int64_t ks[4] = {k.stride(0), k.stride(1), k.stride(2), k.stride(3)};
  const int64_t vs[4] = {v.stride(0), v.stride(1), v.stride(2), v.stride(3)};
  // Under torch.use_deterministic_algorithms(True) take the fixed-order path (the fused kernel
  // adds dQ contributions with reduce-adds in timing-dependent order).
  const auto backward_fn = at::globalContext().deterministicAlgorithms()
                               ? tt_attn_backward_bf16_deterministic
                               : tt_attn_backward_bf16;
  const tt_attn_status st = backward_fn(
      q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, dO.data_ptr(), O.data_ptr(),
      lse.data_ptr<float>(), B, H, Tq, Tk, TT_ATTN_HEAD_DIM, past_len, dq.data_ptr(),
      dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), ws_bytes, static_cast<void*>(stream.stream()));
  TORCH_CHECK(st == TT_ATTN_OK, "tt_attn_backward_bf16 failed: ", tt_attn_status_string(st),
              ": ", tt_attn_last_error());
  return {dq, dk, dv};
}

// Fused RoPE + KV-cache append (tt_rope_append_bf16). `position` is either a Python int or an
// int64 CUDA tensor with one element (read on the device, for captured decode steps).
torch::Tensor rope_append(const torch::Tensor& qkv, const torch::Tensor& cos,
                          const torch::Tensor& sin, const pybind11::object& position,
                          torch::Tensor cache_k, torch::Tensor cache_v) {
  TORCH_CHECK(qkv.is_cuda() && cos.is_cuda() && sin.is_cuda() && cache_k.is_cuda() &&
                  cache_v.is_cuda(), "rope_append: all tensors must be CUDA tensors");
  for (const torch::Tensor* t : {&cos, &sin, static_cast<const torch::Tensor*>(&cache_k),
                                 static_cast<const torch::Tensor*>(&cache_v)})
    TORCH_CHECK(t->device() == qkv.device(), "rope_append: all tensors must be on the same device");
  TORCH_CHECK(qkv.scalar_type() == at::kBFloat16 && cache_k.scalar_type() == at::kBFloat16 &&
                  cache_v.scalar_type() == at::kBFloat16, "rope_append: qkv and caches must be bf16");
  TORCH_CHECK(cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat,
              "rope_append: cos/sin tables must be float32");
  TORCH_CHECK(qkv.dim() == 5 && qkv.size(2) == 3 && qkv.size(4) == TT_ATTN_HEAD_DIM &&
                  qkv.is_contiguous(), "rope_append: qkv must be a contiguous [B, T, 3, H, 64] tensor");
  TORCH_CHECK(cos.dim() == 2 && cos.size(1) == TT_ATTN_HEAD_DIM / 2 && cos.is_contiguous() &&
                  sin.sizes() == cos.sizes() && sin.is_contiguous(),
              "rope_append: cos/sin must be contiguous [L, 32] tables");
  const int64_t B = qkv.size(0), T = qkv.size(1), H = qkv.size(3);
  for (const torch::Tensor* c : {&cache_k, &cache_v})
    TORCH_CHECK(c->dim() == 4 && c->size(0) == B && c->size(1) == H &&
                    c->size(3) == TT_ATTN_HEAD_DIM && c->stride(3) == 1,
                "rope_append: caches must be [B, H, capacity, 64] with contiguous rows");
  TORCH_CHECK(cache_v.size(2) == cache_k.size(2), "rope_append: caches must have equal capacity");
  int64_t pos = 0;
  const int64_t* pos_dev = nullptr;
  torch::Tensor pos_t;
  if (pybind11::isinstance<pybind11::int_>(position)) {
    pos = position.cast<int64_t>();
  } else {
    pos_t = position.cast<torch::Tensor>();
    TORCH_CHECK(pos_t.is_cuda() && pos_t.device() == qkv.device() &&
                    pos_t.scalar_type() == at::kLong && pos_t.numel() == 1,
                "rope_append: a tensor position must be a one-element int64 CUDA tensor");
    pos_dev = pos_t.data_ptr<int64_t>();
  }
  const c10::cuda::CUDAGuard device_guard(qkv.device());
  auto q_out = torch::empty({B, H, T, TT_ATTN_HEAD_DIM}, qkv.options());
  const int64_t ks[4] = {cache_k.stride(0), cache_k.stride(1), cache_k.stride(2), 1};
  const int64_t vs[4] = {cache_v.stride(0), cache_v.stride(1), cache_v.stride(2), 1};
  auto stream = c10::cuda::getCurrentCUDAStream(qkv.get_device());
  const tt_attn_status st = tt_rope_append_bf16(
      qkv.data_ptr(), B, T, H, cos.data_ptr<float>(), sin.data_ptr<float>(), cos.size(0), pos,
      pos_dev, q_out.data_ptr(), cache_k.data_ptr(), ks, cache_v.data_ptr(), vs, cache_k.size(2),
      static_cast<void*>(stream.stream()));
  TORCH_CHECK(st == TT_ATTN_OK, "tt_rope_append_bf16 failed: ", tt_attn_status_string(st), ": ",
              tt_attn_last_error());
  return q_out;
}

// QKV projection + RoPE + KV-cache append in one kernel (tt_qkv_rope_append_bf16). `hidden`
// is the normalised hidden state [B, T, dim]; `w_qkv` the layer's [3 * H * 64, dim] weight;
// `position` as for rope_append.
torch::Tensor qkv_rope_append(const torch::Tensor& hidden, const torch::Tensor& w_qkv,
                              const torch::Tensor& cos, const torch::Tensor& sin,
                              const pybind11::object& position, torch::Tensor cache_k,
                              torch::Tensor cache_v) {
  for (const torch::Tensor* t : {&hidden, &w_qkv, &cos, &sin,
                                 static_cast<const torch::Tensor*>(&cache_k),
                                 static_cast<const torch::Tensor*>(&cache_v)}) {
    TORCH_CHECK(t->is_cuda(), "qkv_rope_append: all tensors must be CUDA tensors");
    TORCH_CHECK(t->device() == hidden.device(),
                "qkv_rope_append: all tensors must be on the same device");
  }
  TORCH_CHECK(hidden.scalar_type() == at::kBFloat16 && w_qkv.scalar_type() == at::kBFloat16 &&
                  cache_k.scalar_type() == at::kBFloat16 && cache_v.scalar_type() == at::kBFloat16,
              "qkv_rope_append: hidden, w_qkv and the caches must be bf16");
  TORCH_CHECK(cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat,
              "qkv_rope_append: cos/sin tables must be float32");
  TORCH_CHECK(hidden.dim() == 3 && hidden.is_contiguous(),
              "qkv_rope_append: hidden must be a contiguous [B, T, dim] tensor");
  const int64_t B = hidden.size(0), T = hidden.size(1), dim = hidden.size(2);
  TORCH_CHECK(w_qkv.dim() == 2 && w_qkv.is_contiguous() && w_qkv.size(1) == dim &&
                  w_qkv.size(0) % (3 * TT_ATTN_HEAD_DIM) == 0,
              "qkv_rope_append: w_qkv must be a contiguous [3 * H * 64, dim] weight");
  const int64_t H = w_qkv.size(0) / (3 * TT_ATTN_HEAD_DIM);
  TORCH_CHECK(cos.dim() == 2 && cos.size(1) == TT_ATTN_HEAD_DIM / 2 && cos.is_contiguous() &&
                  sin.sizes() == cos.sizes() && sin.is_contiguous(),
              "qkv_rope_append: cos/sin must be contiguous [L, 32] tables");
  for (const torch::Tensor* c : {&cache_k, &cache_v})
    TORCH_CHECK(c->dim() == 4 && c->size(0) == B && c->size(1) == H &&
                    c->size(3) == TT_ATTN_HEAD_DIM && c->stride(3) == 1,
                "qkv_rope_append: caches must be [B, H, capacity, 64] with contiguous rows");
  TORCH_CHECK(cache_v.size(2) == cache_k.size(2),
              "qkv_rope_append: caches must have equal capacity");
  int64_t pos = 0;
  const int64_t* pos_dev = nullptr;
  torch::Tensor pos_t;
  if (pybind11::isinstance<pybind11::int_>(position)) {
    pos = position.cast<int64_t>();
  } else {
    pos_t = position.cast<torch::Tensor>();
    TORCH_CHECK(pos_t.is_cuda() && pos_t.device() == hidden.device() &&
                    pos_t.scalar_type() == at::kLong && pos_t.numel() == 1,
                "qkv_rope_append: a tensor position must be a one-element int64 CUDA tensor");
    pos_dev = pos_t.data_ptr<int64_t>();
  }
  const c10::cuda::CUDAGuard device_guard(hidden.device());
  auto q_out = torch::empty({B, H, T, TT_ATTN_HEAD_DIM}, hidden.options());
  const int64_t ks[4] = {cache_k.stride(0), cache_k.stride(1), cache_k.stride(2), 1};
  const int64_t vs[4] = {cache_v.stride(0), cache_v.stride(1), cache_v.stride(2), 1};
  auto stream = c10::cuda::getCurrentCUDAStream(hidden.get_device());
  const tt_attn_status st = tt_qkv_rope_append_bf16(
      hidden.data_ptr(), B, T, dim, w_qkv.data_ptr(), H, cos.data_ptr<float>(),
      sin.data_ptr<float>(), cos.size(0), pos, pos_dev, q_out.data_ptr(), cache_k.data_ptr(), ks,
      cache_v.data_ptr(), vs, cache_k.size(2), static_cast<void*>(stream.stream()));
  TORCH_CHECK(st == TT_ATTN_OK, "tt_qkv_rope_append_bf16 failed: ", tt_attn_status_string(st),
              ": ", tt_attn_last_error());
  return q_out;
}

// ------------------------------------------------------------------ speculative decoding
// Uninitialised CUDA tensor without a trip through the dispatcher: these calls are as short as a
// launch, and every allocation's host time shows.
torch::Tensor new_cuda(at::IntArrayRef sizes, at::ScalarType dtype, const c10::Device& device) {
  return at::detail::empty_cuda(sizes, dtype, device, std::nullopt);
}

// int32 copy of an index tensor where it is not one already; int64 values are clamped into int32,
// so that none wraps into a valid index.
torch::Tensor index32(const torch::Tensor& x, const torch::Tensor& like, const char* what) {
  TORCH_CHECK(x.defined() && x.is_cuda() && x.device() == like.device(), what,
              " must be a CUDA tensor on the same device as the other inputs");
  TORCH_CHECK(x.scalar_type() == at::kInt || x.scalar_type() == at::kLong, what,
              " must be int32 or int64");
  if (x.scalar_type() == at::kInt) return x.is_contiguous() ? x : x.contiguous();
  return x.clamp(std::numeric_limits<int32_t>::min(), std::numeric_limits<int32_t>::max())
      .to(at::kInt)
      .contiguous();
}

// [N] (one tree) or [B, N] parents as int32; returns the row stride the C ABI takes.
torch::Tensor tree_parents(const torch::Tensor& parents, const torch::Tensor& like, int64_t B,
                           int64_t N, int64_t* stride) {
  torch::Tensor p = index32(parents, like, "parents");
  TORCH_CHECK((p.dim() == 1 && p.size(0) == N) ||
                  (p.dim() == 2 && p.size(0) == B && p.size(1) == N),
              "parents must have shape [N] or [B, N]");
  *stride = p.dim() == 2 ? N : 0;
  return p;
}

void check_sm100(const torch::Tensor& x) {
  const auto* props = at::cuda::getDeviceProperties(x.get_device());
  TORCH_CHECK(props->major == 10,
              "the bf16 attention kernels require an sm_100 GPU (compute capability 10.x); "
              "found SM", props->major, props->minor);
}

struct Strides {
  int64_t s[4];
  explicit Strides(const torch::Tensor& x) : s{x.stride(0), x.stride(1), x.stride(2), x.stride(3)} {}
};

// Attention of a tree of drafted tokens over a cache (tt_attn_tree_forward_bf16).
std::tuple<torch::Tensor, torch::Tensor> tree_attention(
    torch::Tensor q, torch::Tensor tree_k, torch::Tensor tree_v, torch::Tensor cache_k,
    torch::Tensor cache_v, torch::Tensor parents, std::optional<torch::Tensor> cache_lens,
    bool with_lse) {
  for (const torch::Tensor* t : {&q, &tree_k, &tree_v, &cache_k, &cache_v}) {
    TORCH_CHECK(t->defined() && t->is_cuda(), "tree_attention: all inputs must be CUDA tensors");
    TORCH_CHECK(t->device() == q.device(),
                "tree_attention: all inputs must be on the same device");
    TORCH_CHECK(t->scalar_type() == at::kBFloat16,
                "tree_attention: q, the tree's K/V and the caches must be bf16");
    TORCH_CHECK(t->layout() == at::kStrided && t->dim() == 4,
                "tree_attention: q, the tree's K/V and the caches must be strided 4D tensors");
    TORCH_CHECK(t->size(3) == TT_ATTN_HEAD_DIM,
                "tree_attention currently supports only head_dim=64");
    TORCH_CHECK(t->size(0) == q.size(0), "tree_attention: all inputs must have the same batch size");
  }
  TORCH_CHECK(!(at::GradMode::is_enabled() &&
                (q.requires_grad() || tree_k.requires_grad() || tree_v.requires_grad() ||
                 cache_k.requires_grad() || cache_v.requires_grad())),
              "tree_attention has no backward; call it under no_grad");
  const int64_t B = q.size(0), Hq = q.size(1), N = q.size(2), Hkv = cache_k.size(1),
                C = cache_k.size(2);
  TORCH_CHECK(B > 0 && Hq > 0 && N > 0 && Hkv > 0 && C > 0,
              "tree_attention: batch, heads, nodes and cache capacity must be positive");
  TORCH_CHECK(Hq % Hkv == 0, "tree_attention: q heads must be a multiple of the K/V heads");
  TORCH_CHECK(N <= TT_ATTN_TREE_MAX_NODES, "tree_attention: at most 256 nodes per tree");
  TORCH_CHECK(cache_v.sizes() == cache_k.sizes(),
              "tree_attention: the K and V caches must have the same shape");
  TORCH_CHECK(tree_k.size(1) == Hkv && tree_k.size(2) == N && tree_v.sizes() == tree_k.sizes(),
              "tree_attention: the tree's K and V must have shape [B, kv_heads, N, 64]");
  if (cache_lens.has_value())
    TORCH_CHECK(cache_lens->defined() && cache_lens->dim() == 1 && cache_lens->size(0) == B,
                "tree_attention: cache_lens must have shape [B]");
  const c10::cuda::CUDAGuard device_guard(q.device());
  check_sm100(q);
  int64_t parents_stride = 0;
  parents = tree_parents(parents, q, B, N, &parents_stride);
  torch::Tensor lens;
  if (cache_lens.has_value()) lens = index32(*cache_lens, q, "cache_lens");
  auto stream = c10::cuda::getCurrentCUDAStream(q.get_device());
  q = aligned_contiguous(q);
  tree_k = aligned_contiguous(tree_k);
  tree_v = aligned_contiguous(tree_v);
  cache_k = aligned_contiguous(cache_k);
  cache_v = aligned_contiguous(cache_v);
  auto o = new_cuda({B, Hq, N, TT_ATTN_HEAD_DIM}, at::kBFloat16, q.device());
  torch::Tensor lse;
  if (with_lse) lse = new_cuda({B, Hq, N}, at::kFloat, q.device());
  const size_t ws_bytes = tt_attn_tree_workspace_size(B, Hq, Hkv, N, C);
  torch::Tensor ws;
  if (ws_bytes > 0)
    ws = new_cuda({static_cast<int64_t>(ws_bytes)}, at::kByte, q.device());
  const Strides qs(q), tks(tree_k), tvs(tree_v), cks(cache_k), cvs(cache_v);
  const tt_attn_status st = tt_attn_tree_forward_bf16(
      q.data_ptr(), qs.s, tree_k.data_ptr(), tks.s, tree_v.data_ptr(), tvs.s, cache_k.data_ptr(),
      cks.s, cache_v.data_ptr(), cvs.s, B, Hq, Hkv, N, C, TT_ATTN_HEAD_DIM,
      parents.data_ptr<int32_t>(), parents_stride,
      lens.defined() ? lens.data_ptr<int32_t>() : nullptr, o.data_ptr(),
      with_lse ? lse.data_ptr<float>() : nullptr, ws_bytes > 0 ? ws.data_ptr() : nullptr, ws_bytes,
      static_cast<void*>(stream.stream()));
  TORCH_CHECK(st == TT_ATTN_OK, "tt_attn_tree_forward_bf16 failed: ", tt_attn_status_string(st),
              ": ", tt_attn_last_error());
  return {o, lse};
}

// Walk of a token tree with given random numbers (tt_attn_tree_verify_f32).
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> tree_verify(
    torch::Tensor tokens, torch::Tensor parents, torch::Tensor target_probs,
    torch::Tensor uniforms, std::optional<torch::Tensor> draft_probs) {
  TORCH_CHECK(target_probs.defined() && target_probs.is_cuda(),
              "verify_tree: all inputs must be CUDA tensors");
  TORCH_CHECK(target_probs.scalar_type() == at::kFloat && target_probs.dim() == 3,
              "verify_tree: target_probs must be a float32 [B, N, V] tensor");
  const int64_t B = target_probs.size(0), N = target_probs.size(1), V = target_probs.size(2);
  TORCH_CHECK(B > 0 && N > 0 && V > 0, "verify_tree: batch, nodes and vocabulary must be positive");
  TORCH_CHECK(N <= TT_ATTN_TREE_MAX_NODES, "verify_tree: at most 256 nodes per tree");
  TORCH_CHECK(V <= TT_ATTN_TREE_MAX_VOCAB,
              "verify_tree: at most ", TT_ATTN_TREE_MAX_VOCAB, " tokens in the vocabulary");
  for (const torch::Tensor* t : {&tokens, &uniforms})
    TORCH_CHECK(t->defined() && t->is_cuda() && t->device() == target_probs.device(),
                "verify_tree: all inputs must be CUDA tensors on the same device");
  TORCH_CHECK(tokens.dim() == 2 && tokens.size(0) == B && tokens.size(1) == N &&
                  (tokens.scalar_type() == at::kLong || tokens.scalar_type() == at::kInt),
              "verify_tree: tokens must be an int64 or int32 [B, N] tensor");
  TORCH_CHECK(uniforms.dim() == 2 && uniforms.size(0) == B && uniforms.size(1) == N &&
                  uniforms.scalar_type() == at::kFloat,
              "verify_tree: uniforms must be a float32 [B, N] tensor");
  const bool dense = draft_probs.has_value();
  if (dense)
    TORCH_CHECK(draft_probs->defined() && draft_probs->is_cuda() &&
                    draft_probs->device() == target_probs.device() &&
                    draft_probs->scalar_type() == at::kFloat &&
                    draft_probs->sizes() == target_probs.sizes(),
                "verify_tree: draft_probs must be a float32 [B, N, V] tensor on the same device");
  const c10::cuda::CUDAGuard device_guard(target_probs.device());
  check_sm100(target_probs);
  int64_t parents_stride = 0;
  parents = tree_parents(parents, target_probs, B, N, &parents_stride);
  if (tokens.scalar_type() != at::kLong) tokens = tokens.to(at::kLong);
  if (!tokens.is_contiguous()) tokens = tokens.contiguous();
  if (!uniforms.is_contiguous()) uniforms = uniforms.contiguous();
  // Rows are read in place when their values are adjacent; other views are copied.
  if (V > 1 && target_probs.stride(2) != 1) target_probs = target_probs.contiguous();
  torch::Tensor dp;
  if (dense)
    dp = V > 1 && draft_probs->stride(2) != 1 ? draft_probs->contiguous() : *draft_probs;
  auto path = new_cuda({B, N}, at::kInt, target_probs.device());
  auto counts = new_cuda({B}, at::kInt, target_probs.device());
  auto next = new_cuda({B}, at::kLong, target_probs.device());
  auto stream = c10::cuda::getCurrentCUDAStream(target_probs.get_device());
  const tt_attn_status st = tt_attn_tree_verify_f32(
      tokens.data_ptr<int64_t>(), parents.data_ptr<int32_t>(), parents_stride,
      target_probs.data_ptr<float>(), target_probs.stride(0), target_probs.stride(1),
      dense ? dp.data_ptr<float>() : nullptr, dense ? dp.stride(0) : 0, dense ? dp.stride(1) : 0,
      uniforms.data_ptr<float>(), B, N, V, path.data_ptr<int32_t>(), counts.data_ptr<int32_t>(),
      next.data_ptr<int64_t>(), static_cast<void*>(stream.stream()));
  TORCH_CHECK(st == TT_ATTN_OK, "tt_attn_tree_verify_f32 failed: ", tt_attn_status_string(st), ": ",
              tt_attn_last_error());
  return {path, counts, next};
}

// One list of the commit's per-layer tensors (caches or trees): all checks of a tensor in one pass,
// since there are four tensors a layer on every step.
struct LayerTensors {
  std::vector<torch::Tensor> t;
  bool in_place = true;  // equal strides, and every tensor can be read (and written) where it is
};

LayerTensors layer_tensors(const pybind11::list& list, c10::Device* device) {
  LayerTensors out;
  out.t.reserve(list.size());
  const bool grad = at::GradMode::is_enabled();
  for (const pybind11::handle item : list) {
    TORCH_CHECK(THPVariable_Check(item.ptr()), "commit_path: caches and trees must be tensors");
    const torch::Tensor& x = THPVariable_Unpack(item.ptr());
    TORCH_CHECK(x.is_cuda(), "commit_path: all inputs must be CUDA tensors");
    if (out.t.empty() && device->is_cpu()) *device = x.device();
    TORCH_CHECK(x.device() == *device, "commit_path: all inputs must be on the same device");
    TORCH_CHECK(x.scalar_type() == at::kBFloat16 && x.layout() == at::kStrided && x.dim() == 4,
                "commit_path: caches and trees must be strided 4D bf16 tensors");
    TORCH_CHECK(x.size(3) == TT_ATTN_HEAD_DIM, "commit_path currently supports only head_dim=64");
    TORCH_CHECK_NOT_IMPLEMENTED(
        !(grad && x.requires_grad()),
        "commit_path writes the caches in place and has no backward; call it under no_grad");
    out.t.push_back(x);
    const torch::Tensor& first = out.t.front();
    TORCH_CHECK(x.sizes() == first.sizes(),
                "commit_path: all caches, and all trees, must have the same shape");
    bool same = readable_in_place(x);
    for (int64_t d = 0; d < 4; ++d) same = same && (x.size(d) == 1 || x.stride(d) == first.stride(d));
    out.in_place = out.in_place && same;
  }
  return out;
}

// Append of the accepted path to the caches of all layers (tt_attn_tree_commit_bf16).
torch::Tensor tree_commit(const pybind11::list& cache_k, const pybind11::list& cache_v,
                          const pybind11::list& tree_k, const pybind11::list& tree_v,
                          torch::Tensor path, torch::Tensor counts, torch::Tensor cache_lens) {
  const size_t L = cache_k.size();
  TORCH_CHECK(L > 0 && cache_v.size() == L && tree_k.size() == L && tree_v.size() == L,
              "commit_path: the caches and the trees must have the same, positive number of layers");
  TORCH_CHECK(!at::autocast::is_autocast_enabled(at::kCUDA),
              "commit_path does not support AMP/autocast yet");
  c10::Device device(at::kCPU);
  LayerTensors c[2] = {layer_tensors(cache_k, &device), layer_tensors(cache_v, &device)};
  LayerTensors t[2] = {layer_tensors(tree_k, &device), layer_tensors(tree_v, &device)};
  const torch::Tensor& first = c[0].t[0];
  const int64_t B = first.size(0), H = first.size(1), C = first.size(2), N = t[0].t[0].size(2);
  TORCH_CHECK(B > 0 && H > 0 && C > 0 && N > 0, "commit_path: sizes must be positive");
  TORCH_CHECK(c[1].t[0].sizes() == first.sizes(),
              "commit_path: all caches must have the same shape");
  for (int i = 0; i < 2; ++i) {
    TORCH_CHECK(c[i].in_place,
                "commit_path: the caches need equal strides, a unit last stride, other strides in "
                "multiples of 8 elements and 16-byte aligned bases (they are written in place)");
    const torch::Tensor& x = t[i].t[0];
    TORCH_CHECK(x.size(0) == B && x.size(1) == H && x.size(2) == N,
                "commit_path: the trees must have shape [B, kv_heads, N, 64]");
  }
  TORCH_CHECK(path.defined() && path.dim() == 2 && path.size(0) == B && path.size(1) > 0,
              "commit_path: path must have shape [B, P]");
  TORCH_CHECK(counts.defined() && counts.dim() == 1 && counts.size(0) == B && cache_lens.defined() &&
                  cache_lens.dim() == 1 && cache_lens.size(0) == B,
              "commit_path: counts and cache_lens must have shape [B]");
  const c10::cuda::CUDAGuard device_guard(device);
  check_sm100(first);
  path = index32(path, first, "path");
  counts = index32(counts, first, "counts");
  cache_lens = index32(cache_lens, first, "cache_lens");
  for (LayerTensors& x : t)
    if (!x.in_place)
      for (torch::Tensor& y : x.t) y = y.clone(at::MemoryFormat::Contiguous);
  auto new_lens = new_cuda({B}, at::kInt, device);
  std::vector<void*> ptr(4 * L);
  for (size_t l = 0; l < L; ++l) {
    ptr[l] = c[0].t[l].data_ptr();
    ptr[L + l] = c[1].t[l].data_ptr();
    ptr[2 * L + l] = t[0].t[l].data_ptr();
    ptr[3 * L + l] = t[1].t[l].data_ptr();
  }
  const Strides cks(first), cvs(c[1].t[0]), tks(t[0].t[0]), tvs(t[1].t[0]);
  auto stream = c10::cuda::getCurrentCUDAStream(device.index());
  const tt_attn_status st = tt_attn_tree_commit_bf16(
      ptr.data(), cks.s, ptr.data() + L, cvs.s, ptr.data() + 2 * L, tks.s, ptr.data() + 3 * L, tvs.s,
      static_cast<int64_t>(L), B, H, N, C, TT_ATTN_HEAD_DIM, path.data_ptr<int32_t>(), path.size(1),
      counts.data_ptr<int32_t>(), cache_lens.data_ptr<int32_t>(), new_lens.data_ptr<int32_t>(),
      static_cast<void*>(stream.stream()));
  TORCH_CHECK(st == TT_ATTN_OK, "tt_attn_tree_commit_bf16 failed: ", tt_attn_status_string(st), ": ",
              tt_attn_last_error());
  return new_lens;
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("attention_forward", &attention_forward,
        "BF16 causal attention forward on sm_100a (returns O and natural-log FP32 LSE)",
        pybind11::arg("q"), pybind11::arg("k"), pybind11::arg("v"),
        pybind11::arg("past_len") = 0, pybind11::arg("segment_ids") = pybind11::none(),
        pybind11::arg("kv_lens") = pybind11::none());
  m.def("attention_backward", &attention_backward,
        "BF16 causal attention backward on sm_100a (preprocess, dQ, dK/dV); returns dq, dk, dv",
        pybind11::arg("q"), pybind11::arg("k"), pybind11::arg("v"), pybind11::arg("dO"),
        pybind11::arg("O"), pybind11::arg("lse"), pybind11::arg("past_len") = 0,
        pybind11::arg("segment_ids") = pybind11::none());
  m.def("rope_append", &rope_append,
        "Fused RoPE on q/k of a [B, T, 3, H, 64] QKV projection + KV-cache append; returns rope(q)",
        pybind11::arg("qkv"), pybind11::arg("cos"), pybind11::arg("sin"),
        pybind11::arg("position"), pybind11::arg("cache_k"), pybind11::arg("cache_v"));
  m.def("qkv_rope_append", &qkv_rope_append,
        "QKV projection + RoPE on q/k + KV-cache append in one kernel; returns rope(q)",
        pybind11::arg("hidden"), pybind11::arg("w_qkv"), pybind11::arg("cos"),
        pybind11::arg("sin"), pybind11::arg("position"), pybind11::arg("cache_k"),
        pybind11::arg("cache_v"));
  m.def("tree_attention", &tree_attention,
        "Attention of a tree of drafted tokens over a KV cache; returns O and (with_lse) LSE",
        pybind11::arg("q"), pybind11::arg("tree_k"), pybind11::arg("tree_v"),
        pybind11::arg("cache_k"), pybind11::arg("cache_v"), pybind11::arg("parents"),
        pybind11::arg("cache_lens") = pybind11::none(), pybind11::arg("with_lse") = true);
  m.def("tree_verify", &tree_verify,
        "Walk of a drafted token tree with given random numbers; returns path, counts, next tokens",
        pybind11::arg("tokens"), pybind11::arg("parents"), pybind11::arg("target_probs"),
        pybind11::arg("uniforms"), pybind11::arg("draft_probs") = pybind11::none());
  m.def("tree_commit", &tree_commit,
        "Append of the accepted path's K/V rows to the caches of all layers; returns new lengths",
        pybind11::arg("cache_k"), pybind11::arg("cache_v"), pybind11::arg("tree_k"),
        pybind11::arg("tree_v"), pybind11::arg("path"), pybind11::arg("counts"),
        pybind11::arg("cache_lens"));
  m.attr("HEAD_DIM") = TT_ATTN_HEAD_DIM;
  m.attr("ABI_VERSION") = TT_ATTN_ABI_VERSION;
}
