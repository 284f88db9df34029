"""Fused operators around the attention call (the caller side of the hot path)."""
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


def qkv_norm_rope(qkv, q_weight, k_weight, cos, sin, position=0, eps=1e-6, kv_heads=None):
    """RMS norm of every query and key head of a fused projection, and the position rotation, in one pass;
    returns ``(q, k, v)`` as ``student.attention`` takes them (with as many K/V as query heads: shared ones go there
    after ``repeat_interleave(Hq // Hkv, 1)``).

    ``qkv`` is BF16 ``[B, T, 3, H, 64]``, or ``[B, T, Hq + 2 Hkv, 64]`` (query, key, value heads) with
    ``kv_heads=Hkv``; ``q_weight`` / ``k_weight`` ``[64]``, BF16 or FP32 (both None: the rotation alone);
    ``cos`` / ``sin`` FP32 ``[L, 32]`` tables, a row per position. ``position`` is the first position (an int),
    or an int64 CUDA tensor read on the device: one element, ``[B]`` (a first position for each sequence) or
    ``[B, T]`` (one for each token: packed documents; ``student.attention`` has no mask between them).

    A head x becomes ``n = x * rsqrt(mean(x^2) + eps) * weight``, its adjacent pairs turned by the table row; FP32
    throughout, rounded once. ``q`` ``[B, Hq, T, 64]`` and ``k`` ``[B, Hkv, T, 64]`` are contiguous, ``v`` is a view of
    ``qkv``. Rows whose position on the device is outside the table are zero and set the range bit of the
    device status (``tt_attn_device_status``).

    Differentiable in ``qkv`` and the weights: the backward reads q's, k's and v's gradients and writes ``qkv``'s
    whole, in one kernel; the weights' gradients are summed in a fixed order. There is no second derivative and no
    forward-mode one (``NotImplementedError``). Forward and backward can be captured
    together in a CUDA graph; while an autograd graph of the same leaves from the default stream lives, that is refused.
    The reference has no such norm (its blocks norm the hidden state only, model.py:46-76).
    """
    return load_attention_extension().qkv_norm_rope(qkv, q_weight, k_weight, cos, sin, position, eps,
                                                    kv_heads)
