"""Speculative decoding over the KV cache: attention of a drafted token tree, its verification, and
the append of the accepted path.

One pass of the target over a tree of N drafted tokens replaces up to depth + 1 single-token steps,
each of which would stream the weights and the cache once. The drafted tokens' K/V rows stay
outside the cache (as the views of the fused projection that a model computes anyway) until the
walk has decided which of them to keep.

A tree is given by ``parents``: int32 or int64 CUDA ``[N]`` (one tree for the batch) or ``[B, N]``.
``parents[n]`` is a lower index, or -1 for a root; node 0 is the last committed token, whose K/V row
is not in the cache yet. A node whose chain of parents does not reach -1 over strictly lower indices
(-2, say) is not in use: padding of a smaller tree. ``N`` is at most 256.

The reference has no counterpart: it generates one token at a time (tiny_transformer/generate.py).
"""
from __future__ import annotations

import torch

from ._extension import load_attention_extension


def _guard(name, tensors):
    grad = torch.is_grad_enabled()
    for x in tensors:
        if not x.is_cuda:
            raise RuntimeError(f"{name} requires CUDA tensors")
        if grad and x.requires_grad:
            raise NotImplementedError(f"{name} has no backward; call it under torch.no_grad()")
    if torch.is_autocast_enabled("cuda"):
        raise RuntimeError(f"{name} does not support AMP/autocast yet")


def tree_attention(q, tree_k, tree_v, cache_k, cache_v, parents, cache_lens=None):
    """Attention of the tree's nodes; returns O ``[B, Hq, N, 64]`` BF16, contiguous.

    ``q`` is ``[B, Hq, N, 64]``, ``tree_k`` / ``tree_v`` the nodes' own rows ``[B, Hkv, N, 64]``,
    ``cache_k`` / ``cache_v`` ``[B, Hkv, C, 64]``, all BF16; ``Hq`` is a multiple of ``Hkv`` and
    query head h reads K/V head ``h // (Hq // Hkv)``. Node n of sequence b sees cache rows
    ``[0, cache_lens[b])`` (int32/int64 CUDA ``[B]``, clamped to ``[0, C]``; None: all C rows) and
    its chain of parents, itself included; scale 1/8, FP32 softmax, its weights rounded to BF16 for the
    product with V. A node not in use gets O = 0.
    Rows that a node does not see never change its output, whatever they hold.

    Strided views are read in place under the rules of ``student.attention``; others are copied.
    Runs on the current CUDA stream; inference only.
    """
    _guard("tree_attention", (q, tree_k, tree_v, cache_k, cache_v))
    output, _ = load_attention_extension().tree_attention(q, tree_k, tree_v, cache_k, cache_v,
                                                          parents, cache_lens, False)
    return output


def tree_attention_with_lse(q, tree_k, tree_v, cache_k, cache_v, parents, cache_lens=None):
    """Like :func:`tree_attention` but returns ``(O, LSE)``; LSE is FP32 ``[B, Hq, N]``, natural log
    (-inf for a node not in use)."""
    _guard("tree_attention_with_lse", (q, tree_k, tree_v, cache_k, cache_v))
    return load_attention_extension().tree_attention(q, tree_k, tree_v, cache_k, cache_v, parents,
                                                     cache_lens, True)


def verify_tree(tokens, parents, target_probs, uniforms, draft_probs=None):
    """Walk of the tree with given random numbers (speculative sampling).

    ``tokens`` int64 ``[B, N]``; ``target_probs`` FP32 ``[B, N, V]``: row n is the target's
    distribution of the token after node n; ``draft_probs`` likewise the distribution from which
    n's children were drawn, independently (None: they were chosen, not drawn); ``uniforms`` FP32
    ``[B, N]`` in ``[0, 1)``: entry n decides node n, entry 0 draws the next token.

    From node 0 on, the current node's children are tried in index order. A child with token t is
    accepted with probability ``min(1, p(t) / q(t))``; otherwise p becomes ``max(p - q, 0)``,
    renormalised, for the next child. When none is accepted the next token is drawn from what is
    left of p, so that path and next token are distributed as the target's own samples.

    Returns ``(path, counts, next_tokens)``: int32 ``[B, N]`` accepted nodes from node 0 on, then
    -1; int32 ``[B]`` how many (0 where node 0 is not a root); int64 ``[B]`` (-1 where counts is 0 or
    no token has any weight).

    Probabilities are weighed as whole multiples of 2^-36, so the result depends on no order of
    summation: the same inputs give the same walk on any split of the work. Uniforms that are 2^-24
    apart, as ``torch.rand`` draws them, resolve the next token's probabilities to 2^-24.
    """
    return load_attention_extension().tree_verify(tokens, parents, target_probs, uniforms,
                                                  draft_probs)


def commit_path(cache_k, cache_v, tree_k, tree_v, path, counts, cache_lens):
    """Append the accepted path's K/V rows to the caches, in place, all layers in one launch.

    ``cache_k`` / ``cache_v`` are one tensor ``[B, Hkv, C, 64]`` or a list of one per layer, ``tree_k``
    / ``tree_v`` ``[B, Hkv, N, 64]`` likewise, all BF16; ``path`` ``[B, P]`` and ``counts`` ``[B]`` as
    :func:`verify_tree` returns them, ``cache_lens`` ``[B]`` the lengths before the append. Row i of
    sequence b goes from tree row ``path[b, i]`` to cache row ``cache_lens[b] + i``.

    Returns the new lengths, int32 ``[B]``. Rows past the capacity and path entries outside the
    tree are skipped and set the range bit of the device status (``tt_attn_device_status``). The length
    counts the row of such a path entry although it is not written: after that status the rows appended
    to the sequence must not be used.
    """
    lists = [x if isinstance(x, list) else list(x) if isinstance(x, tuple) else [x]
             for x in (cache_k, cache_v, tree_k, tree_v)]
    # Four tensors a layer: device, gradient and shape are checked natively, in one pass.
    return load_attention_extension().tree_commit(*lists, path, counts, cache_lens)
