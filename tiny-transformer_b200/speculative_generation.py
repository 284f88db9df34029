"""Speculative generation: a draft model proposes a tree of tokens, the target runs once over it.

Around one step the three operators of ``operators.speculative`` run together as a server would run
them: ``tree_attention`` in every layer of both models (the drafted tokens' K/V rows stay outside the
caches), ``verify_tree`` on the target's and the draft's probabilities, ``commit_path`` on all layers of
both caches. Sequences accept different numbers of tokens, so lengths and positions are per sequence
and live on the device.

The sampled tokens are distributed as the target's own (``temperature`` > 0), or are its greedy choice
(``temperature`` 0: the draft's most probable tokens as children, a one-hot target). The reference
generates one token at a time (tiny_transformer/generate.py:9-29).
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

from .generation import Decoder, KVCache, rms_norm, rope


class TokenTree:
    """A fixed tree shape in level order: ``branching[d]`` children of every node at depth d.

    ``parents`` is the int32 tensor ``[N]`` that the operators take, ``depths`` each node's depth,
    ``levels`` the (first, last + 1) node of each depth.
    """

    def __init__(self, branching, device="cpu"):
        if any(k <= 0 for k in branching):
            raise ValueError("every branching factor must be positive")
        parents, depths, self.levels = [-1], [0], [(0, 1)]
        for depth, k in enumerate(branching):
            first, last = self.levels[-1]
            parents += [n for n in range(first, last) for _ in range(k)]
            depths += [depth + 1] * (k * (last - first))
            self.levels.append((last, len(parents)))
        self.branching = tuple(branching)
        self.size, self.depth = len(parents), len(branching)
        self.parents = torch.tensor(parents, dtype=torch.int32, device=device)
        self.depths = torch.tensor(depths, dtype=torch.long, device=device)

    def to(self, device):
        return TokenTree(self.branching, device)


def _ops():
    from .operators import speculative
    return speculative


def allocate(model: Decoder, cache: KVCache):
    """Allocate every layer's storage of a cache that may not have seen a token yet."""
    cfg = model.config
    proto = model.embedding.new_empty((cache.batch_size, cfg.n_heads, 1, cfg.head_dim))
    for layer in range(cfg.n_layers):
        cache._storage(layer, proto, proto)


def forward_tree(model: Decoder, ids, tree_parents, depths, cache: KVCache, lens, ops=None):
    """One pass of ``model`` over the drafted tokens ``ids`` ``[B, N]``: logits ``[B, N, V]`` and the
    nodes' K and V rows of every layer, ``[B, H, N, 64]`` each. Node n of sequence b is at position
    ``lens[b] + depths[n]``, which has to stay below ``max_seq_len``, and sees cache rows
    ``[0, lens[b])`` and its own branch; the cache is not changed."""
    ops = ops or _ops()
    cfg = model.config
    batch, nodes = ids.shape
    positions = lens.long()[:, None] + depths                       # [B, N]
    cos, sin = model.rope_cos[positions][:, None], model.rope_sin[positions][:, None]
    x = F.embedding(ids, model.embedding)
    keys, values = [], []
    for layer, block in enumerate(model.blocks):
        h = rms_norm(x, block.attn_norm, cfg.norm_eps)
        qkv = F.linear(h, block.qkv).view(batch, nodes, 3, cfg.n_heads, cfg.head_dim)
        q, k, v = (t.transpose(1, 2) for t in qkv.unbind(dim=2))
        q, k = rope(q, cos, sin), rope(k, cos, sin)
        attended = ops.tree_attention(q, k, v, cache.keys[layer], cache.values[layer], tree_parents,
                                      lens)
        x = block.finish(x, attended)
        keys.append(k)
        values.append(v)
    return model.logits(x), keys, values


def _probabilities(logits, temperature):
    """FP32 next-token distributions; at temperature 0 all weight on the most probable token."""
    if temperature == 0:
        return F.one_hot(logits.argmax(-1), logits.shape[-1]).float()
    return torch.softmax(logits.float() / temperature, dim=-1)


def propose(draft: Decoder, root, tree: TokenTree, cache: KVCache, lens, temperature, generator=None,
            ops=None):
    """Draft tokens of the whole tree, level by level: ``(tokens [B, N], q [B, N, V] or None, keys,
    values)``. Children are drawn from the draft's distribution at their parent, independently, and q
    holds those distributions; at temperature 0 they are its most probable tokens and q is None."""
    batch, vocab = root.shape[0], draft.config.vocab_size
    tokens = torch.zeros(batch, tree.size, dtype=torch.long, device=root.device)
    tokens[:, 0] = root
    q = (None if temperature == 0 else
         torch.zeros(batch, tree.size, vocab, dtype=torch.float32, device=root.device))
    for (first, last), (nxt, end), k in zip(tree.levels, tree.levels[1:], tree.branching):
        logits, _, _ = forward_tree(draft, tokens[:, :last], tree.parents[:last], tree.depths[:last],
                                    cache, lens, ops)
        level = logits[:, first:last]
        if temperature == 0:
            children = level.topk(k, dim=-1).indices
        else:
            # Any distribution may propose as long as the walk is told which: a row without one (logits
            # that are not finite; sampling from it would be a device-side assertion) becomes uniform.
            rows = _probabilities(level, temperature).nan_to_num_(nan=1 / vocab)
            q[:, first:last] = rows
            children = torch.multinomial(rows.flatten(0, 1), k, replacement=True, generator=generator)
        tokens[:, nxt:end] = children.reshape(batch, end - nxt)
    # All nodes once more: the leaves' K/V rows belong to the path too.
    _, keys, values = forward_tree(draft, tokens, tree.parents, tree.depths, cache, lens, ops)
    return tokens, q, keys, values


@torch.inference_mode()
def generate_speculative(model: Decoder, draft: Decoder, prompt, new_tokens: int, branching=(3, 2, 1),
                         temperature: float = 1.0, generator=None, ops=None):
    """Generate ``new_tokens`` per sequence after ``prompt`` ``[B, T]`` with a draft model.

    ``branching`` is the tree's shape (children per node at each depth). Returns ``(tokens
    [B, new_tokens], stats)``; ``stats["steps"]`` target passes and ``stats["accepted"]`` the mean
    number of tokens a pass yielded. Raises RuntimeError where the target's logits are not finite and
    no token can be drawn from them. ``ops`` replaces the operators (a test runs the host logic on CPU
    with it).
    """
    if new_tokens <= 0:
        raise ValueError("new_tokens must be positive")
    if temperature < 0:
        raise ValueError("temperature must not be negative")
    if model.config.vocab_size != draft.config.vocab_size:
        raise ValueError("the draft needs the target's vocabulary")
    ops = ops or _ops()
    device = prompt.device
    batch, time = prompt.shape
    tree = TokenTree(branching, device)
    capacity = time + new_tokens + tree.depth
    for m in (model, draft):
        if capacity > m.config.max_seq_len:
            raise ValueError("sequence exceeds model max_seq_len")
    caches = [m.new_cache(batch, capacity) for m in (model, draft)]
    for m, cache in zip((model, draft), caches):
        allocate(m, cache)
        if time > 1:
            m(prompt[:, :-1], cache=cache, last_only=True)
    # The last token of the prompt is the first root: it is in no cache yet.
    lens = torch.full((batch,), time - 1, dtype=torch.int32, device=device)
    root = prompt[:, -1]
    # The last column takes what is not kept.
    out = torch.zeros(batch, new_tokens + 1, dtype=torch.long, device=device)
    have = torch.zeros(batch, dtype=torch.int32, device=device)
    column = torch.arange(tree.size, device=device)
    steps, yielded = 0, 0
    while True:
        tokens, q, dk, dv = propose(draft, root, tree, caches[1], lens, temperature, generator, ops)
        logits, tk, tv = forward_tree(model, tokens, tree.parents, tree.depths, caches[0], lens, ops)
        uniforms = torch.rand(batch, tree.size, device=device, generator=generator)
        path, counts, nxt = ops.verify_tree(tokens, tree.parents, _probabilities(logits, temperature),
                                            uniforms, q)
        # Not past the last token that is asked for: a finished sequence stands still while the others
        # go on, with its length at most time - 1 + new_tokens and its nodes inside the tables.
        kept = torch.minimum(counts, new_tokens - have)
        ops.commit_path(caches[1].keys, caches[1].values, dk, dv, path, kept, lens)
        lens = ops.commit_path(caches[0].keys, caches[0].values, tk, tv, path, kept, lens)
        # The accepted tokens after the root, then the drawn one: counts of them.
        step = tokens.gather(1, path.clamp(min=0).long()).roll(-1, dims=1)
        step = torch.where(column[None] == counts[:, None].long() - 1, nxt[:, None], step)
        at = torch.where(column[None] < kept[:, None], have[:, None] + column[None], new_tokens)
        out.scatter_(1, at, step)
        have = have + kept
        # The drawn token of a path kept whole is output, and the next root: -1 (the target's row has no
        # weight, so its logits are not finite) must not reach the embedding.
        whole = kept == counts
        root = torch.where(whole, nxt, root)
        steps += 1
        done, undrawn = torch.stack([have.sum(), (whole & (nxt < 0)).sum()]).tolist()
        if undrawn:
            raise RuntimeError("no token can be drawn: the target's logits are not finite")
        yielded = done
        if done == batch * new_tokens:
            break
    return out[:, :new_tokens].clone(), {"steps": steps, "accepted": yielded / (batch * steps)}
