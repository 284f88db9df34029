"""KV cache held in 4 bits: append (with the head norm and the rotation in the same pass), read back, attention.

A cache is a uint8 CUDA tensor ``[B, Hkv, blocks, 576]``, one for the keys and one for the values of a layer; its
capacity is ``16 * blocks`` rows (tokens). A block holds 16 rows of 64 features as 512 bytes of e2m1 codes and 64
bytes of scales, one for 16 features (36 bytes a row against 128 in BF16; the exact layout is in
``include/tt_attention.h``). A value is its code times its scale. Rows are quantised as they are written:
the scale is the group's largest magnitude over 6, rounded to 4 significant bits (2^-14 to 10240; fewer bits down to
2^-17, that is for groups whose largest value is below 3.7e-4, and zero below 2.3e-5), codes go to the
nearest value, of two to the one with the even code. A group with a NaN reads back as NaN; larger values saturate.

The reference has no counterpart: its cache has the model's type (tiny_transformer/model.py:11-43).
"""
from __future__ import annotations

import torch

from ._extension import load_attention_extension

BLOCK_ROWS = 16
BLOCK_BYTES = 576
MAX_QUERIES = 16


def new_cache(batch, kv_heads, capacity, device="cuda"):
    """A zeroed cache for ``capacity`` rows (rounded up to whole blocks of 16)."""
    if batch <= 0 or kv_heads <= 0 or capacity <= 0:
        raise ValueError("a 4-bit cache needs a positive batch, heads and capacity")
    blocks = -(-capacity // BLOCK_ROWS)
    return torch.zeros(batch, kv_heads, blocks, BLOCK_BYTES, dtype=torch.uint8, device=device)


def append(qkv, cos, sin, position, cache_k, cache_v, q_weight=None, k_weight=None, eps=1e-6):
    """Norm, rotation and quantised append of a fused projection, in one kernel; returns q ``[B, Hq, T, 64]``.

    ``qkv``, ``cos`` / ``sin``, the weights and ``eps`` as in :func:`fused.qkv_norm_rope` (weights None: no norm), with
    as many K/V heads as the caches have. Token t of sequence b goes to row ``position + t`` of the caches:
    ``position`` is an int, or an int64 CUDA tensor with one element or one for each sequence, read on the
    device (a captured step, sequences of different lengths). The keys are quantised from their BF16 values as
    64 bits give them (rounded by way of FP32), so the bytes do not depend on the order of a sum; other rows stay as
    they are.
    Rows outside the cache or the tables are not written, their q is zero, and the range bit of the device
    status is set (``tt_attn_device_status``). Views whose blocks overlap, in one cache or between the two, are
    refused; the halves of one ``[B, 2, Hkv, blocks, 576]`` tensor are fine. Runs on the current CUDA stream; inference
    only.
    """
    return load_attention_extension().cache4_append(qkv, cos, sin, position, cache_k, cache_v, q_weight,
                                                    k_weight, eps)


def read(cache_k, cache_v, start, rows):
    """Rows ``start`` to ``start + rows - 1`` of both caches as BF16 ``[B, Hkv, rows, 64]`` (exact).

    ``start`` is an int, or an int64 CUDA tensor with one element or one for each sequence; rows outside the cache
    then read as zero and set the range bit of the device status.
    """
    return load_attention_extension().cache4_read(cache_k, cache_v, start, rows)


def attention(q, cache_k, cache_v, kv_lens=None):
    """Attention of the last T <= 16 tokens of each sequence over a 4-bit cache; returns O ``[B, Hq, T, 64]`` BF16.

    ``q`` is BF16 ``[B, Hq, T, 64]``, Hq a multiple of the caches' heads: query head h reads K/V head
    ``h // (Hq // Hkv)``. ``kv_lens`` (int32/int64 CUDA ``[B]``, clamped to the capacity; None: all rows) counts
    the T tokens' own rows: query t sees rows ``j < kv_lens[b] - (T - 1 - t)``. Scale 1/8, FP32 softmax, its weights
    rounded to half precision for the product with V; the codes are used as they are, never expanded in
    memory. A query that sees no row gets O = 0. Rows that a query does not see never change its output, whatever
    they hold. Longer prompts read their rows back (:func:`read`) for ``student.attention``, which wants as many K/V as
    query heads (``repeat_interleave`` of shared ones).
    Runs on the current CUDA stream; inference only.
    """
    return load_attention_extension().cache4_attention(q, cache_k, cache_v, kv_lens)


def attention_with_lse(q, cache_k, cache_v, kv_lens=None):
    """Like :func:`attention` but returns ``(O, LSE)``; LSE is FP32 ``[B, Hq, T]``, natural log (-inf for a query
    that sees no row)."""
    return load_attention_extension().cache4_attention_with_lse(q, cache_k, cache_v, kv_lens)
