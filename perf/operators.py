"""Timed cases of the speculative-decoding operators, with their plain forms.

The operators are reached through ``tiny_transformer_b200.operators.speculative``:

* ``tree_attention`` / ``tree_attention_with_lse``: attention of a tree of drafted tokens over a
  KV cache (each node sees the cached prefix, its ancestors and itself);
* ``verify_tree``: walks the tree with given random numbers and target / draft probabilities,
  returning the accepted path and the next token;
* ``commit_path``: appends the accepted path's K/V rows to the caches of all layers.

With ``own`` false, ``run`` computes the same with elementary torch operations. ``exact`` computes
it once more, in 64 bits, from the definitions.
"""
import math

import numpy as np
import torch

own = False

HEAD_DIM = 64
ONE = 2.0 ** 36  # fixed-point unit of the verification's weights
UNUSED = -2      # parent of a node that is not in use

# ------------------------------------------------------------------------------- the cases


def listed():
    def tree(name, B, Hq, Hkv, N, C, lo, hi, fan, ragged=False, lse=False):
        return dict(name=name, op="tree", B=B, Hq=Hq, Hkv=Hkv, N=N, C=C, lo=lo, hi=hi, fan=fan,
                    ragged=ragged, lse=lse)

    def verify(name, B, N, V, fan, dense, ragged=False):
        return dict(name=name, op="verify", B=B, N=N, V=V, fan=fan, dense=dense, ragged=ragged)

    def commit(name, L, B, H, N, C, lo, hi):
        return dict(name=name, op="commit", L=L, B=B, H=H, N=N, C=C, lo=lo, hi=hi)

    return [
        # One user, a chain of 8 drafted tokens over a short cache: latency.
        tree("tree_b1_n8_c512", 1, 12, 12, 8, 512, 128, 512, 1),
        # The small serving batch of the framework's decode benchmark, a binary tree.
        tree("tree_b8_n16_c512", 8, 12, 12, 16, 512, 256, 512, 2),
        # A tree of one node: the plain decode step of a speculative server with drafting off.
        tree("tree_b32_n1_c1024", 32, 12, 12, 1, 1024, 512, 1024, 1, lse=True),
        # The large serving batch of the decode benchmark, cache lengths 1024 to 8192.
        tree("tree_b64_n16_c8192", 64, 12, 12, 16, 8192, 1024, 8192, 3),
        # Large trees over caches of the model's own maximum length.
        tree("tree_b32_n64_c4096", 32, 12, 12, 64, 4096, 1024, 4096, 4),
        # Shared K/V heads, odd sizes, another tree for each sequence with unused nodes.
        tree("tree_b3_g3_n37_c20001", 3, 12, 4, 37, 20001, 9000, 20001, 3, ragged=True, lse=True),
        # One user, a chain, the framework's vocabulary: latency.
        verify("verify_b1_n8_v8192", 1, 8, 8192, 1, True),
        # A serving batch, a tree with siblings drawn from the draft's distribution.
        verify("verify_b32_n16_v8192", 32, 16, 8192, 3, True),
        # A draft without probabilities (top tokens), an odd vocabulary, ragged trees.
        verify("verify_b5_n24_v50257_top", 5, 24, 50257, 4, False, ragged=True),
        # A large vocabulary and a large batch of trees.
        verify("verify_b32_n32_v128000", 32, 32, 128000, 2, True),
        # All layers of one user's cache after a step.
        commit("commit_l8_b1_n8_c512", 8, 1, 12, 8, 512, 128, 480),
        # All layers of a serving batch after a step with large trees.
        commit("commit_l8_b32_n64_c512", 8, 32, 12, 64, 512, 64, 448),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "verify", "verify", "commit"])
    if op == "tree":
        Hkv, G = rng.choice([(12, 1), (12, 1), (8, 1), (4, 3), (2, 4), (3, 2), (1, 8)])
        B, N, C = _log_int(rng, 1, 64), _log_int(rng, 1, 64), _log_int(rng, 64, 20001)
        if G * N > 128:
            N = 128 // G
        # No more cache, and no more products, than the largest listed case of each.
        while B > 1 and (B * Hkv * C > 64 * 12 * 4608 or B * Hkv * G * N * C > 32 * 12 * 64 * 2560):
            B = B // 2
        hi = rng.randint(C // 2, C)
        return dict(op=op, B=B, Hq=Hkv * G, Hkv=Hkv, N=N, C=C, lo=rng.randint(0, hi), hi=hi,
                    fan=rng.choice([1, 2, 3, 4]), ragged=rng.random() < 0.5, lse=rng.random() < 0.5)
    if op == "verify":
        B, N, V = _log_int(rng, 1, 32), _log_int(rng, 1, 32), _log_int(rng, 257, 128000)
        return dict(op=op, B=B, N=N, V=V, fan=rng.choice([1, 2, 3, 4]), dense=rng.random() < 0.7,
                    ragged=rng.random() < 0.5)
    N, C = _log_int(rng, 1, 64), _log_int(rng, 96, 512)
    return dict(op=op, L=rng.randint(1, 8), B=_log_int(rng, 1, 32), H=rng.choice([1, 4, 12]), N=N,
                C=C, lo=0, hi=rng.randint(0, C - N))


# ------------------------------------------------------------------------------- inputs


def _lengths(case):
    """B lengths spread evenly over [lo, hi]: the same multiset for every seed."""
    B, lo, hi = case["B"], case["lo"], case["hi"]
    return [lo + int((hi - lo) * (i + 0.5) / B) for i in range(B)]


def _parents(case, rs):
    """[N] int32 for a fan-out-`fan` tree in level order; ragged: [B, N], another random tree for
    each sequence, of another size, the rest unused."""
    B, N, fan = case["B"], case["N"], case["fan"]
    regular = np.array([(n - 1) // fan if n else -1 for n in range(N)], dtype=np.int32)
    if not case["ragged"]:
        return regular
    p = np.empty((B, N), dtype=np.int32)
    for b in range(B):
        for n in range(N):
            p[b, n] = -1 if n == 0 else rs.randint(max(0, n - 2 * fan), n)
        p[b, rs.randint((N + 1) // 2, N + 1):] = UNUSED
    return p


def _bf16(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(torch.bfloat16)


def _caches(gen, B, H, C):
    """[B, H, C, 64] bf16, made in slices (no second copy of a large cache in 32 bits)."""
    out = torch.empty(B, H, C, HEAD_DIM, device="cuda", dtype=torch.bfloat16)
    for b in range(B):
        out[b] = torch.randn(H, C, HEAD_DIM, generator=gen, device="cuda")
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rs = np.random.RandomState(seed % (2 ** 32))
    dev = "cuda"
    B, N = case["B"], case["N"]
    s = dict(op=case["op"])
    if case["op"] == "tree":
        Hq, Hkv, C = case["Hq"], case["Hkv"], case["C"]
        # q, k and v of the step as the views of one fused projection, which they are in a model.
        qkv = _bf16(gen, B, N, Hq + 2 * Hkv, HEAD_DIM)
        q, k, v = (t.transpose(1, 2) for t in qkv.split([Hq, Hkv, Hkv], dim=2))
        s.update(q=q, tree_k=k, tree_v=v, cache_k=_caches(gen, B, Hkv, C),
                 cache_v=_caches(gen, B, Hkv, C), lse=case["lse"])
        s["parents"] = torch.from_numpy(_parents(case, rs)).to(dev)
        s["cache_lens"] = torch.from_numpy(
            rs.permutation(np.array(_lengths(case), dtype=np.int32))).to(dev)
    elif case["op"] == "verify":
        V = case["V"]
        parents = torch.from_numpy(_parents(case, rs)).to(dev)
        logits = torch.randn(B, N, V, generator=gen, device=dev).mul_(3)
        s["target_probs"] = torch.softmax(logits, -1)
        # The draft is the target's distribution with an error of its own.
        logits.add_(torch.randn(B, N, V, generator=gen, device=dev), alpha=0.7)
        logits = torch.softmax(logits, -1)
        up = parents.clamp(min=0).long().expand(B, N)
        if case["dense"]:  # tokens drawn from the distribution at the parent
            race = torch.empty(N, V, device=dev)
            tok = [(logits[b][up[b]] / race.exponential_(generator=gen)).argmax(-1) for b in range(B)]
            s["draft_probs"] = logits
        else:              # the k-th child of a node is its k-th most probable token
            k = min(N, V)
            top = logits.topk(k, dim=-1).indices
            order = (up[:, :, None] == up[:, None, :]).tril(-1).sum(-1).clamp(max=k - 1)
            tok = [top[b][up[b], order[b]] for b in range(B)]
            s["draft_probs"] = None
        s["tokens"] = torch.stack(tok)
        s["parents"] = parents
        s["uniforms"] = torch.rand(B, N, generator=gen, device=dev)
    else:
        L, H, C = case["L"], case["H"], case["C"]
        s["cache_k"] = [_caches(gen, B, H, C) for _ in range(L)]
        s["cache_v"] = [_caches(gen, B, H, C) for _ in range(L)]
        kv = [_bf16(gen, B, N, 2, H, HEAD_DIM) for _ in range(L)]
        s["tree_k"] = [t[:, :, 0].transpose(1, 2) for t in kv]
        s["tree_v"] = [t[:, :, 1].transpose(1, 2) for t in kv]
        path = np.full((B, N), -1, dtype=np.int32)
        counts = rs.permutation(np.array(_counts(case), dtype=np.int32))
        for b in range(B):
            path[b, :counts[b]] = np.sort(rs.permutation(N)[:counts[b]])
            path[b, 0] = 0
        s["path"] = torch.from_numpy(path).to(dev)
        s["counts"] = torch.from_numpy(counts).to(dev)
        s["cache_lens"] = torch.from_numpy(
            rs.permutation(np.array(_lengths(case), dtype=np.int32))).to(dev)
    return s


def _counts(case):
    """Accepted nodes (the root among them) of each sequence: 1 to about a tree's depth."""
    top = min(case["N"], 8)
    return [1 + i % top for i in range(case["B"])] if case["B"] > 1 else [(top + 1) // 2]


# ------------------------------------------------------------------------------- one pass


def run(state):
    s = state
    if own:
        from __graft_entry__ import import_package
        import_package()
        from tiny_transformer_b200.operators import speculative
        if s["op"] == "tree":
            call = speculative.tree_attention_with_lse if s["lse"] else speculative.tree_attention
            return call(s["q"], s["tree_k"], s["tree_v"], s["cache_k"], s["cache_v"], s["parents"],
                        s["cache_lens"])
        if s["op"] == "verify":
            return speculative.verify_tree(s["tokens"], s["parents"], s["target_probs"],
                                           s["uniforms"], s["draft_probs"])
        lens = speculative.commit_path(s["cache_k"], s["cache_v"], s["tree_k"], s["tree_v"],
                                       s["path"], s["counts"], s["cache_lens"])
        return [lens, s["cache_k"], s["cache_v"]]
    if s["op"] == "tree":
        return _plain_tree(s)
    if s["op"] == "verify":
        return _plain_verify(s)
    return _plain_commit(s)


def _ancestors(parents):
    """[B, N, N] bool: node m is n itself or an ancestor of n, by doubling the ancestor relation;
    rows of unused nodes are empty."""
    N = parents.shape[-1]
    at = torch.arange(N, device=parents.device)
    ok = (parents >= -1) & (parents < at)
    step = ((parents[..., None] == at) & ok[..., None]) | torch.eye(N, dtype=torch.bool, device=parents.device)
    reach = step.float()
    for _ in range(max(1, (N - 1).bit_length())):
        reach = (torch.matmul(reach, reach) > 0).float()
    # In use: no node on the chain has a parent that is neither -1 nor a lower index.
    used = torch.matmul(reach, (~ok).float()[..., None]) == 0
    return (reach > 0) & used


def _plain_tree(s):
    q, C = s["q"].float(), s["cache_k"].shape[2]
    B, Hq, N, _ = q.shape
    Hkv = s["cache_k"].shape[1]
    inside = (torch.arange(C, device=q.device) < s["cache_lens"][:, None])[:, None, :, None]
    zero = torch.zeros((), device=q.device)
    k = torch.cat([torch.where(inside, s["cache_k"].float(), zero), s["tree_k"].float()], 2)
    v = torch.cat([torch.where(inside, s["cache_v"].float(), zero), s["tree_v"].float()], 2)
    tree = _ancestors(s["parents"].expand(B, N))
    used = tree.any(-1)
    cached = inside[:, 0, :, 0]                                            # [B, C]
    mask = torch.cat([cached[:, None] & used[..., None], tree], -1)[:, None, None]
    scores = torch.matmul(q.reshape(B, Hkv, -1, HEAD_DIM), k.transpose(2, 3)).mul_(0.125)
    scores = scores.view(B, Hkv, Hq // Hkv, N, C + N).masked_fill_(~mask, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    top = torch.where(used[:, None, None, :, None], top, zero)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, Hkv, -1, C + N), v).view(B, Hkv, -1, N, HEAD_DIM)
    o = torch.where(total > 0, o / total, zero).to(torch.bfloat16).reshape(B, Hq, N, HEAD_DIM)
    if not s["lse"]:
        return o
    return o, (top + total.log()).reshape(B, Hq, N)


def _plain_verify(s):
    tokens, p, q, u = s["tokens"], s["target_probs"], s["draft_probs"], s["uniforms"]
    B, N, V = p.shape
    parents = s["parents"].expand(B, N)
    row = torch.arange(B, device=p.device)
    fixed = lambda x: x.double().mul(ONE).floor().long()  # noqa: E731
    cur = torch.zeros(B, dtype=torch.long, device=p.device)
    count = torch.ones_like(cur)
    order = torch.zeros(B, N, dtype=torch.long, device=p.device)
    tried = torch.zeros_like(cur)                       # children rejected at the current node
    total = torch.full_like(cur, int(ONE))
    r = fixed(p[:, 0])
    # A node's children come after it, in the order in which they are tried, so one walk over the
    # nodes in index order visits each child when its parent's turn has come.
    for c in range(1, N):
        here = parents[:, c] == cur
        t = tokens[:, c]
        qc = torch.nn.functional.one_hot(t, V).float() if q is None else q[row, cur]
        qt, pt = qc[row, t], p[row, cur, t]
        first = u[:, c] * qt < pt
        later = u[:, c].double() * qt.double() * total.double() < r[row, t].double()
        take = here & torch.where(tried == 0, first, later)
        drop = here & ~take
        left = (r - (qc.double() * total.double()[:, None]).floor().long()).clamp(min=0)
        r = torch.where(drop[:, None], left, torch.where(take[:, None], fixed(p[:, c]), r))
        total = torch.where(drop, r.sum(-1), torch.where(take, int(ONE), total))
        tried = torch.where(take, 0, tried + drop)
        cur = torch.where(take, c, cur)
        order[:, c] = torch.where(take, count, 0)
        count = count + take
    r = torch.where((r.sum(-1) > 0)[:, None], r, fixed(p[row, cur]))
    run_sum = r.cumsum(-1)
    goal = (u[:, 0].double() * run_sum[:, -1].double()).floor().long()
    nxt = (run_sum <= goal[:, None]).sum(-1)
    path = torch.full((B, N + 1), -1, dtype=torch.int32, device=p.device)
    at = torch.arange(N, device=p.device, dtype=torch.int32).expand(B, N)
    path.scatter_(1, torch.where(order > 0, order, N), at)
    path[:, 0] = 0
    return path[:, :N].contiguous(), count.int(), nxt


def _plain_commit(s):
    N, counts = s["path"].shape[1], s["counts"]
    i = torch.arange(N, device=counts.device)
    i = torch.where(i < counts[:, None], i, 0)          # past the path: its first row once more
    b = torch.arange(len(counts), device=counts.device)[:, None]
    src, dst = s["path"].gather(1, i).long(), (s["cache_lens"][:, None] + i).long()
    for cache, tree in zip(s["cache_k"] + s["cache_v"], s["tree_k"] + s["tree_v"]):
        cache[b, :, dst] = tree[b, :, src]
    return [s["cache_lens"] + counts, s["cache_k"], s["cache_v"]]


# ------------------------------------------------------------------------------- 64 bits


def _chains(parents):
    """For each node of one tree the list of its ancestors and itself; [] for an unused node."""
    out = []
    for n in range(len(parents)):
        chain, m = [], n
        while 0 <= m and parents[m] < m and parents[m] >= -1:
            chain.append(m)
            m = int(parents[m])
        out.append(chain if m == -1 else [])
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "commit":
        return None  # copies: nothing is computed
    B, N = case["B"], case["N"]
    parents = np.broadcast_to(s["parents"].cpu().numpy(), (B, N))
    if case["op"] == "verify":
        return _exact_verify(s, parents)
    Hq, Hkv = case["Hq"], case["Hkv"]
    G = Hq // Hkv
    o = torch.zeros(B, Hq, N, HEAD_DIM, dtype=torch.float64, device="cuda")
    lse = torch.full((B, Hq, N), float("-inf"), dtype=torch.float64, device="cuda")
    lens = s["cache_lens"].tolist()
    for b in range(B):
        chains = _chains(parents[b])
        for h in range(Hkv):
            heads = slice(h * G, (h + 1) * G)
            qb = s["q"][b, heads].double() / math.sqrt(HEAD_DIM)           # [G, N, 64]
            kc, vc = (s[x][b, h, :lens[b]].double() for x in ("cache_k", "cache_v"))
            kt, vt = (s[x][b, h].double() for x in ("tree_k", "tree_v"))
            sc, st = qb @ kc.T, qb @ kt.T
            see = torch.zeros(N, N, dtype=torch.bool)
            for n, chain in enumerate(chains):
                see[n, chain] = True
            st = st.masked_fill(~see.to(st.device), float("-inf"))
            both = torch.cat([sc, st], -1)
            use = [n for n in range(N) if chains[n]]
            lse[b, heads, use] = torch.logsumexp(both[:, use], -1)
            w = torch.exp(both[:, use] - lse[b, heads, use][..., None])
            o[b, heads, use] = w[..., :lens[b]] @ vc + w[..., lens[b]:] @ vt
    return (o, lse) if case["lse"] else o


def _exact_verify(s, parents):
    """Whole numbers, from the definition: one sequence at a time, one child at a time."""
    B, N = parents.shape
    tokens, u = s["tokens"].cpu().numpy(), s["uniforms"].cpu().numpy()
    path, count, nxt = np.full((B, N), -1, np.int32), np.zeros(B, np.int32), np.zeros(B, np.int64)
    for b in range(B):
        cur, taken = 0, [0]
        while True:
            p = s["target_probs"][b, cur].cpu().numpy().astype(np.float64)
            q = None if s["draft_probs"] is None else s["draft_probs"][b, cur].cpu().numpy().astype(np.float64)
            r, total, accepted = np.floor(p * ONE).astype(np.int64), int(ONE), None
            for k, c in enumerate([c for c in range(cur + 1, N) if parents[b, c] == cur]):
                t = tokens[b, c]
                qc = np.zeros_like(p) if q is None else q
                if q is None:
                    qc[t] = 1.0
                if k == 0:
                    hit = np.float32(u[b, c]) * np.float32(qc[t]) < np.float32(p[t])
                else:
                    hit = float(u[b, c]) * qc[t] * float(total) < float(r[t])
                if hit:
                    accepted = c
                    break
                r = np.maximum(r - np.floor(qc * float(total)).astype(np.int64), 0)
                total = int(r.sum())
            if accepted is None:
                if r.sum() == 0:
                    r = np.floor(p * ONE).astype(np.int64)
                goal = math.floor(float(u[b, 0]) * float(r.sum()))
                nxt[b] = np.searchsorted(np.cumsum(r), goal, side="right")
                break
            cur = accepted
            taken.append(cur)
        path[b, :len(taken)] = taken
        count[b] = len(taken)
    return path, count, nxt


# ------------------------------------------------------------------------------- least work


def work(case):
    """Each input that the pass needs read once, each output written once."""
    B, N = case["B"], case["N"]
    if case["op"] == "tree":
        Hq, Hkv, rows = case["Hq"], case["Hkv"], sum(_lengths(case))
        q_o = 2 * B * Hq * N * HEAD_DIM * 2 + (4 * B * Hq * N if case["lse"] else 0)
        kv = 2 * HEAD_DIM * 2 * Hkv * (rows + B * N)
        depth = 1 + (N - 1 if case["fan"] == 1 else int(math.log(max(N, 1), case["fan"])))
        return dict(bytes=q_o + kv + 4 * (B + N),
                    flops=4 * HEAD_DIM * Hq * (N * rows + B * N * min(N, depth)))
    if case["op"] == "verify":
        # The target's row where the walk ends, the draft's too (a child was rejected there, or
        # not: counted as read in half of the sequences), and a few values for each node.
        rows = 1.5 if case["dense"] else 1.0
        return dict(bytes=int(B * case["V"] * 4 * rows) + B * N * 28, flops=3 * B * case["V"])
    rows = sum(_counts(case))
    return dict(bytes=2 * 2 * HEAD_DIM * 2 * case["L"] * case["H"] * rows + 4 * B * (N + 3), flops=0)
