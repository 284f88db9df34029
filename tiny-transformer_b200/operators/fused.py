"""Fused operators around the attention call (the caller side of the hot path)."""
import torch
from torch.autograd.function import once_differentiable

from ._extension import load_attention_extension


def rope_append(qkv, cos, sin, position, cache_k, cache_v):
    """RoPE on q and k of a fused QKV projection plus the KV-cache append, in one kernel.

    ``qkv`` is the contiguous ``[B, T, 3, H, 64]`` BF16 output of the QKV linear (the
    reference reshapes it the same way, model.py:60); ``cos`` / ``sin`` are FP32 ``[L, 32]``
    tables indexed by position; ``position`` is the first position (an int, or a one-element
    int64 CUDA tensor read on the device). Writes rope(k) and v into rows ``position + t`` of
    the ``[B, H, C, 64]`` caches and returns rope(q) as ``[B, H, T, 64]``. Bit-exact with the
    reference's bf16 ``rope`` (reference.py:30-34) followed by ``KVCache.update``
    (model.py:29-41).
    """
    return load_attention_extension().rope_append(qkv, cos, sin, position, cache_k, cache_v)


def qkv_rope_append(hidden, w_qkv, cos, sin, position, cache_k, cache_v):
    """The QKV projection of a decoder layer with RoPE and the KV-cache append in its epilogue.

    ``hidden`` is the normalised hidden state ``[B, T, dim]`` (BF16, contiguous), ``w_qkv`` the
    layer's ``[3 * H * 64, dim]`` weight (the reference's ``Block.qkv``). Equivalent to
    ``rope_append(F.linear(hidden, w_qkv).view(B, T, 3, H, 64), ...)`` with the projection
    accumulated in FP32 inside the kernel and never written to memory (model.py:59-67); returns
    rope(q) as ``[B, H, T, 64]``.
    """
    return load_attention_extension().qkv_rope_append(hidden, w_qkv, cos, sin, position,
                                                      cache_k, cache_v)


class _QkvNormRope(torch.autograd.Function):
    """Norm and rotation forward and backward through the native module. v is a view of qkv, so that its
    gradient goes into the one dqkv that the backward kernel writes."""

    @staticmethod
    def forward(ctx, qkv, q_weight, k_weight, cos, sin, position, eps, kv_heads):
        q, k = load_attention_extension().qkv_norm_rope(qkv, q_weight, k_weight, cos, sin, position,
                                                        eps, kv_heads)
        ctx.save_for_backward(qkv, q_weight, k_weight, cos, sin,
                              position if torch.is_tensor(position) else None)
        ctx.position, ctx.eps, ctx.kv_heads = position if not torch.is_tensor(position) else None, eps, kv_heads
        ctx.set_materialize_grads(False)
        return q, k, _value_heads(qkv, kv_heads)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk, dv):
        qkv, q_weight, k_weight, cos, sin, position = ctx.saved_tensors
        if dq is None and dk is None and dv is None:
            return (None,) * 8
        dqkv, dqw, dkw = load_attention_extension().qkv_norm_rope_backward(
            qkv, q_weight, k_weight, cos, sin, ctx.position if position is None else position, ctx.eps,
            ctx.kv_heads, dq, dk, dv)
        need = ctx.needs_input_grad
        return (dqkv if need[0] else None, dqw if need[1] else None, dkw if need[2] else None,
                None, None, None, None, None)


def _value_heads(qkv, kv_heads):
    """The value heads of a projection as a [B, Hkv, T, 64] view."""
    return (qkv[:, :, 2] if qkv.dim() == 5 else qkv[:, :, qkv.shape[2] - kv_heads:]).transpose(1, 2)


def qkv_norm_rope(qkv, q_weight, k_weight, cos, sin, position=0, eps=1e-6, kv_heads=None):
    """RMS norm of every query and key head of a fused projection, and the position rotation, in one pass;
    returns ``(q, k, v)`` as ``student.attention`` takes them.

    ``qkv`` is BF16 ``[B, T, 3, H, 64]``, or ``[B, T, Hq + 2 Hkv, 64]`` (query, key, value heads) with
    ``kv_heads=Hkv``; ``q_weight`` / ``k_weight`` ``[64]``, BF16 or FP32 (both None: the rotation alone);
    ``cos`` / ``sin`` FP32 ``[L, 32]`` tables, a row per position. ``position`` is the first position (an int),
    or an int64 CUDA tensor read on the device: one element, ``[B]`` (a first position for each sequence) or
    ``[B, T]`` (one for each token: packed documents).

    A head x becomes ``n = x * rsqrt(mean(x^2) + eps) * weight``, its adjacent pairs turned by the table row; FP32
    throughout, rounded once. ``q`` ``[B, Hq, T, 64]`` and ``k`` ``[B, Hkv, T, 64]`` are contiguous, ``v`` is a view of
    ``qkv``. Rows whose position on the device is outside the table are zero and set the range bit of the
    device status (``tt_attn_device_status``).

    Differentiable in ``qkv`` and the weights: the backward reads q's, k's and v's gradients and writes ``qkv``'s
    whole, in one kernel; the weights' gradients are summed in a fixed order. The reference has no such norm (its blocks
    norm the hidden state only, model.py:46-76).
    """
    if not qkv.is_cuda:
        raise RuntimeError("qkv_norm_rope requires CUDA tensors")
    if torch.is_autocast_enabled("cuda"):
        raise RuntimeError("qkv_norm_rope does not support AMP/autocast yet")
    if torch.is_tensor(cos) and (cos.requires_grad or sin.requires_grad) and torch.is_grad_enabled():
        raise NotImplementedError("qkv_norm_rope has no gradient for the cos/sin tables")
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad
                                       for x in (qkv, q_weight, k_weight)):
        return _QkvNormRope.apply(qkv, q_weight, k_weight, cos, sin, position, eps, kv_heads)
    q, k = load_attention_extension().qkv_norm_rope(qkv, q_weight, k_weight, cos, sin, position, eps,
                                                    kv_heads)
    return q, k, _value_heads(qkv, kv_heads)
