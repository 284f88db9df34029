"""Speculative-decoding operators on the GPU against their 64-bit restatements
(oracle/speculative_oracle.py).

Tolerances. bf16 has 8 significand bits: rounding to nearest is within 2^-8 of the value. Tree
attention: P is rounded to bf16 before P.V (2^-8 of each weight), O once at the end (2^-8 of
itself); scores, exponentials and sums are FP32, together below 2^-11 of the weights for the sizes
here. So |O - ref| <= 2^-8 |ref| + (2^-8 + 2^-11) A, A the same average of |v|. LSE: scores are
FP32 sums of 64 products with sum |q k| / 8 below 16, so below 64 * 2^-23 * 16 = 1.2e-4, and below 2^-20
of its value from the logarithm. Verification and commits are whole numbers and copies: equal.
"""
import numpy as np
import pytest
import torch

from oracle import speculative_oracle as oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available() or torch.cuda.get_device_capability()[0] != 10:
        pytest.skip("needs an sm_100 GPU")


@pytest.fixture(scope="module")
def spec():
    from tiny_transformer_b200.operators import speculative
    return speculative


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen).to(torch.bfloat16)


def _tree(rs, N, fan, unused=0):
    p = np.array([-1 if n == 0 else rs.randint(max(0, n - fan), n) for n in range(N)], np.int32)
    if unused:
        p[N - unused:] = -2
    return p


def _case(B, Hq, Hkv, N, C, seed, fan=3, ragged=False):
    gen, rs = torch.Generator().manual_seed(seed), np.random.RandomState(seed)
    t = dict(q=_randn(gen, B, Hq, N, 64), tree_k=_randn(gen, B, Hkv, N, 64),
             tree_v=_randn(gen, B, Hkv, N, 64), cache_k=_randn(gen, B, Hkv, C, 64),
             cache_v=_randn(gen, B, Hkv, C, 64))
    parents = np.stack([_tree(rs, N, fan, rs.randint(0, N // 2 + 1) if ragged else 0)
                        for _ in range(B)])
    return t, parents, rs


def _check(got, lse, t, parents, lens):
    ref, ref_lse, A = oracle.tree_attention(*(t[k].double().numpy() for k in
                                              ("q", "tree_k", "tree_v", "cache_k", "cache_v")),
                                            parents, lens)
    got, lse = got.double().cpu().numpy(), lse.double().cpu().numpy()
    empty = np.isneginf(ref_lse)
    assert (got[empty] == 0).all() and np.isneginf(lse[empty]).all()
    err = np.abs(got - ref)
    assert (err <= 2.0 ** -8 * np.abs(ref) + (2.0 ** -8 + 2.0 ** -11) * A).all(), err.max()
    lerr = np.abs(lse[~empty] - ref_lse[~empty])
    assert (lerr <= 1.2e-4 + 2.0 ** -20 * np.abs(ref_lse[~empty])).all(), lerr.max()


def _run(spec, t, parents, lens, **over):
    d = {k: (over[k] if k in over else v.cuda()) for k, v in t.items()}
    p = torch.from_numpy(np.ascontiguousarray(parents)).cuda()
    n = None if lens is None else torch.as_tensor(lens, dtype=torch.int32).cuda()
    return spec.tree_attention_with_lse(d["q"], d["tree_k"], d["tree_v"], d["cache_k"],
                                        d["cache_v"], p, n)


@pytest.mark.parametrize("B,Hq,Hkv,N,C,lens,ragged", [
    (1, 1, 1, 1, 1, [1], False),              # one node, one cached row
    (2, 2, 2, 1, 200, [0, 200], False),       # nothing cached: a node sees itself
    (3, 2, 2, 8, 129, [1, 128, 129], False),  # tile edges
    (2, 3, 3, 16, 300, [127, 257], False),
    (2, 2, 1, 17, 150, [33, 150], True),      # 34 rows: more than one row tile
    (3, 6, 2, 11, 500, [0, 31, 480], True),   # shared heads, 33 rows
    (2, 8, 1, 5, 90, [64, 90], True),         # 40 rows
    (1, 2, 2, 64, 1000, [999], False),
    (1, 8, 2, 37, 300, [290], True),          # 148 rows: more than one 128-row tile
    (2, 1, 1, 129, 260, [0, 200], True),      # the tree needs two key tiles
    (1, 1, 1, 256, 70, [64], False),          # most nodes
    (1, 2, 1, 200, 40, [40], True),
    (1, 1, 1, 3, 9000, [8999], False),        # a long cache split over CTAs
    (1, 4, 1, 24, 4100, [4097], True),
    (5, 2, 2, 4, 64, [-3, 0, 1, 64, 1000], True),  # lengths are clamped
])
def test_tree_attention_matches_oracle(spec, B, Hq, Hkv, N, C, lens, ragged):
    t, parents, _ = _case(B, Hq, Hkv, N, C, 7 * N + C, ragged=ragged)
    o, lse = _run(spec, t, parents, lens)
    _check(o, lse, t, parents, lens)
    # The same without LSE, and bit for bit the same on a second run.
    d = {k: v.cuda() for k, v in t.items()}
    again = spec.tree_attention(d["q"], d["tree_k"], d["tree_v"], d["cache_k"], d["cache_v"],
                                torch.from_numpy(parents).cuda(), torch.tensor(lens).cuda())
    assert torch.equal(o, again)


@pytest.mark.parametrize("B,Hq,Hkv,N,C,lens,ragged", [
    (2, 4, 4, 24, 70000, [300, 5], True),    # a large capacity: 24 rows in the persistent kernel
    (2, 8, 2, 8, 140000, [1000, 0], False),  # 32 rows of four shared heads
    (1, 2, 2, 40, 4100, [4097], False),      # units shared by CTAs, 40 rows
    (2, 2, 1, 100, 3000, [2999, 10], True),  # 200 rows in two tiles, one short sequence
    (3, 1, 1, 65, 5000, [0, 4990, 129], True),
    (1, 4, 4, 33, 130, [130], False),        # whole units
    (5, 1, 1, 17, 128, [128, 0, 1, 127, 64], True),   # two 16-row tiles, two steps over the tree
    (1, 16, 1, 32, 260, [259], True),        # 512 rows, 32 tiles of one K/V head
])
def test_tree_attention_variants(spec, B, Hq, Hkv, N, C, lens, ragged):
    """Sizes on both sides of the choices between and within the kernels."""
    t, parents, _ = _case(B, Hq, Hkv, N, C, 3 * N + C, ragged=ragged)
    o, lse = _run(spec, t, parents, lens)
    _check(o, lse, t, parents, lens)
    o2, lse2 = _run(spec, t, parents, lens)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("N,C", [(24, 70000), (140, 700)])
def test_masked_places_in_the_persistent_kernel(spec, value, N, C):
    """As above where the persistent kernel runs; 140 nodes span two key tiles. Unused nodes, cached
    rows past the length, and the V rows of leaves in both tiles."""
    lens = [130, 0]
    t, parents, _ = _case(2, 4, 4, N, C, 13, fan=4)
    parents[:, N - 3:] = -2
    want, want_lse = _run(spec, t, parents, lens)
    x = {k: v.clone() for k, v in t.items()}
    for b in range(2):
        x["cache_k"][b, :, lens[b]:] = value
        x["cache_v"][b, :, lens[b]:] = value
    for k in ("q", "tree_k", "tree_v"):
        x[k][:, :, N - 3:] = value
    leaves = [[n for n in range(1, N - 3) if n not in parents[b]] for b in range(2)]
    touched = [{leaves[b][0], leaves[b][-1]} for b in range(2)]
    for b in range(2):
        for n in touched[b]:
            x["tree_v"][b, :, n, 5] = value
    got, lse = _run(spec, x, parents, lens)
    assert torch.equal(lse, want_lse)
    for b in range(2):
        others = [n for n in range(N) if n not in touched[b]]
        assert torch.equal(got[b, :, others], want[b, :, others])
        for n in touched[b]:
            keep = [d for d in range(64) if d != 5]
            assert not torch.isfinite(got[b, :, n, 5]).any()
            # The row's other columns see the finite entries of that V row as before.
            assert torch.equal(got[b, :, n][:, keep], want[b, :, n][:, keep])


@pytest.mark.parametrize("kind", ["chain", "star", "forest", "links"])
def test_tree_shapes(spec, kind):
    """One shared tree [N]: a chain, a star, several roots, and links that end a chain unused."""
    N = 40
    t, _, _ = _case(2, 2, 2, N, 70, 5)
    if kind == "chain":
        one = np.arange(-1, N - 1)
    elif kind == "star":
        one = np.array([-1] + [0] * (N - 1))
    elif kind == "forest":
        one = np.array([-1 if n % 3 == 0 else n - 1 for n in range(N)])
    else:  # self links, links to higher indices, out of range, and nodes below them
        one = np.array([-1] + [n - 1 for n in range(1, N)])
        one[[5, 13, 20, 30]] = [5, 14, 1 << 30, -9]
        one[[8, 16, 23]] = 0
    lens = [70, 3]
    parents = np.broadcast_to(one.astype(np.int32), (2, N))
    d = {k: v.cuda() for k, v in t.items()}
    o, lse = spec.tree_attention_with_lse(
        d["q"], d["tree_k"], d["tree_v"], d["cache_k"], d["cache_v"],
        torch.from_numpy(one.astype(np.int64)).cuda(), torch.tensor(lens, device="cuda"))
    _check(o, lse, t, parents, lens)


def test_int64_parents_outside_int32_are_not_in_use(spec):
    t, _, _ = _case(1, 1, 1, 3, 10, 6)
    d = {k: v.cuda() for k, v in t.items()}
    far = torch.tensor([-1, 1 << 32, (1 << 32) - 1], device="cuda")  # would wrap to 0 and -1
    o, lse = spec.tree_attention_with_lse(d["q"], d["tree_k"], d["tree_v"], d["cache_k"],
                                          d["cache_v"], far, None)
    _check(o, lse, t, np.array([[-1, -2, -2]]), [10])


@pytest.mark.parametrize("G,N", [(1, 12), (1, 30), (3, 16), (2, 64)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -3.38e38])
def test_masked_places_do_not_contribute(spec, value, G, N):
    """Cache rows past the length, unused nodes, and siblings may hold anything."""
    B, C = 2, 300
    lens = [130, 0]
    t, parents, _ = _case(B, 2 * G, 2, N, C, 11, fan=4)
    parents[:, N - 3:] = -2
    want, want_lse = _run(spec, t, parents, lens)
    x = {k: v.clone() for k, v in t.items()}
    for b in range(B):
        x["cache_k"][b, :, lens[b]:] = value
        x["cache_v"][b, :, lens[b]:] = value
    for k in ("q", "tree_k", "tree_v"):
        x[k][:, :, N - 3:] = value
    got, lse = _run(spec, x, parents, lens)
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
    # A leaf's own K and V: only its own row changes.
    leaf = max(n for n in range(N - 3) if n not in parents)
    leaf_b = [n for n in range(N - 3) if n not in parents[0]][-1]
    x["tree_k"][0, :, leaf_b] = value
    x["tree_v"][0, :, leaf_b] = value
    got, lse = _run(spec, x, parents, lens)
    others = [n for n in range(N) if n != leaf_b]
    assert torch.equal(got[:, :, others], want[:, :, others])
    assert torch.equal(lse[:, :, others], want_lse[:, :, others])
    assert leaf is not None


def test_infinite_values_in_view_reach_their_descendants(spec):
    """V of node 1 is +inf: the rows below it are +inf, siblings stay finite."""
    t, _, _ = _case(1, 1, 1, 5, 20, 3)
    one = np.array([[-1, 0, 0, 1, 2]], np.int32)
    want, _ = _run(spec, t, one, [20])
    t["tree_v"][0, 0, 1] = float("inf")
    got, _ = _run(spec, t, one, [20])
    assert torch.isposinf(got[0, 0, [1, 3]]).all()
    assert torch.equal(got[0, 0, [0, 2, 4]], want[0, 0, [0, 2, 4]])


@pytest.mark.parametrize("kind", ["prefix", "token_major", "projection", "feature_stride", "odd"])
def test_layouts(spec, kind):
    """Views read in place and views that have to be copied give the contiguous result."""
    B, H, N, C = 2, 4, 10, 140
    t, parents, _ = _case(B, H, H, N, C, 21)
    lens = [140, 77]
    want = _run(spec, t, parents, lens)
    over = {}
    if kind == "prefix":
        for k in ("cache_k", "cache_v"):
            big = torch.full((B, H, C + 60, 64), float("nan"), dtype=torch.bfloat16, device="cuda")
            big[:, :, :C] = t[k].cuda()
            over[k] = big[:, :, :C]
    elif kind == "token_major":
        for k in t:
            over[k] = t[k].cuda().transpose(1, 2).contiguous().transpose(1, 2)
    elif kind == "projection":
        qkv = torch.cat([t["q"], t["tree_k"], t["tree_v"]], 1).cuda().transpose(1, 2).contiguous()
        for k, x in zip(("q", "tree_k", "tree_v"), qkv.split(H, dim=2)):
            over[k] = x.transpose(1, 2)
    elif kind == "feature_stride":
        for k in t:
            over[k] = t[k].cuda().transpose(2, 3).contiguous().transpose(2, 3)
    else:
        for k in t:
            flat = torch.zeros(t[k].numel() + 1, dtype=torch.bfloat16, device="cuda")
            flat[1:] = t[k].flatten().cuda()
            over[k] = flat[1:].view(t[k].shape)
    got = _run(spec, t, parents, lens, **over)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_offsets_past_32_bits(spec):
    """A cache whose second sequence and last rows start past 2^31 elements."""
    H, N, C, L = 2, 9, 1000, 1000
    t, parents, _ = _case(2, H, H, N, C, 31)
    want = _run(spec, t, parents, [L, L - 1])
    step = (1 << 31) + 64 * 1024
    over = {}
    for i, k in enumerate(("cache_k", "cache_v")):
        store = torch.empty(step + H * C * 64, dtype=torch.bfloat16, device="cuda")
        over[k] = store.as_strided((2, H, C, 64), (step, C * 64, 64, 1))
        over[k].copy_(t[k].cuda())
    got = _run(spec, t, parents, [L, L - 1], **over)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_tree_attention_of_one_node_is_decode(spec):
    """A tree of one node with its row appended is the single-token decode of the framework."""
    from tiny_transformer_b200.operators import student
    B, H, C = 3, 4, 700
    t, parents, _ = _case(B, H, H, 1, C, 41)
    d = {k: v.cuda() for k, v in t.items()}
    with torch.no_grad():
        want, want_lse = student.attention_with_lse(
            d["q"], torch.cat([d["cache_k"], d["tree_k"]], 2),
            torch.cat([d["cache_v"], d["tree_v"]], 2), C)
    o, lse = _run(spec, t, parents, None)
    # Both are within the tolerance above of the exact value; here |v| <= 5 bounds A.
    assert (o.float() - want.float()).abs().max().item() <= 2 * (2.0 ** -8 * 5 + (2.0 ** -8 + 2.0 ** -11) * 5)
    assert (lse - want_lse).abs().max().item() <= 2 * 1.3e-4


def test_runs_on_the_current_stream_and_in_a_graph(spec):
    t, parents, _ = _case(2, 2, 2, 8, 400, 51)
    d = {k: v.cuda() for k, v in t.items()}
    p, lens = torch.from_numpy(parents).cuda(), torch.tensor([400, 250], dtype=torch.int32).cuda()
    want = spec.tree_attention(*d.values(), p, lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = torch.zeros_like(d["q"])
        torch.cuda._sleep(20_000_000)
        late.copy_(d["q"])            # only the side stream orders this before the call
        got = spec.tree_attention(late, *list(d.values())[1:], p, lens)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = spec.tree_attention(*d.values(), p, lens)
    lens.copy_(torch.tensor([0, 399], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    _check(out, spec.tree_attention_with_lse(*d.values(), p, lens)[1], t, parents, [0, 399])


def _bad(spec, **over):
    t, parents, _ = _case(2, 4, 2, 6, 30, 61)
    d = {k: v.cuda() for k, v in t.items()}
    d["parents"], d["cache_lens"] = torch.from_numpy(parents).cuda(), torch.tensor([3, 4]).cuda()
    d.update({k: f(d) for k, f in over.items()})
    return spec.tree_attention(d["q"], d["tree_k"], d["tree_v"], d["cache_k"], d["cache_v"],
                               d["parents"], d["cache_lens"])


@pytest.mark.parametrize("over,error,match", [
    (dict(q=lambda d: d["q"].cpu()), RuntimeError, "CUDA"),
    (dict(q=lambda d: d["q"].float()), RuntimeError, "bf16"),
    (dict(q=lambda d: d["q"][..., :32]), RuntimeError, "head_dim=64"),
    (dict(q=lambda d: d["q"][:, :3]), RuntimeError, "multiple"),
    (dict(q=lambda d: d["q"][:1]), RuntimeError, "batch"),
    (dict(q=lambda d: d["q"][:, :, :5]), RuntimeError, "kv_heads, N, 64"),
    (dict(tree_v=lambda d: d["tree_v"][:, :, :5]), RuntimeError, "kv_heads, N, 64"),
    (dict(cache_v=lambda d: d["cache_v"][:, :, :29]), RuntimeError, "same shape"),
    (dict(cache_k=lambda d: d["cache_k"][0]), RuntimeError, "4D"),
    (dict(cache_k=lambda d: d["cache_k"][:, :, :0], cache_v=lambda d: d["cache_v"][:, :, :0]),
     RuntimeError, "positive"),
    (dict(parents=lambda d: d["parents"][:, :5]), RuntimeError, "parents must have shape"),
    (dict(parents=lambda d: d["parents"].float()), RuntimeError, "int32 or int64"),
    (dict(parents=lambda d: d["parents"].cpu()), RuntimeError, "CUDA"),
    (dict(cache_lens=lambda d: d["cache_lens"][:1]), RuntimeError, "shape"),
    (dict(cache_lens=lambda d: d["cache_lens"].half()), RuntimeError, "int32 or int64"),
    (dict(q=lambda d: d["q"].requires_grad_()), NotImplementedError, "no backward"),
])
def test_tree_attention_refusals(spec, over, error, match):
    with pytest.raises(error, match=match):
        _bad(spec, **over)


def test_tree_attention_refuses_too_many_nodes(spec):
    x = torch.zeros(1, 1, 257, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="256 nodes"):
        spec.tree_attention(x, x, x, x, x, torch.zeros(257, dtype=torch.int32, device="cuda"))


# ------------------------------------------------------------------------------ verification

def _verify_case(B, N, V, seed, dense, fan=3, ragged=False, spread=2.0):
    gen, rs = torch.Generator().manual_seed(seed), np.random.RandomState(seed)
    logits = torch.randn(B, N, V, generator=gen) * spread
    p = torch.softmax(logits, -1)
    q = torch.softmax(logits + torch.randn(B, N, V, generator=gen), -1)
    parents = np.stack([_tree(rs, N, fan, rs.randint(0, N // 2 + 1) if ragged else 0)
                        for _ in range(B)])
    tokens = np.zeros((B, N), np.int64)
    for b in range(B):
        for n in range(1, N):
            w = q[b, max(int(parents[b, n]), 0)].double().numpy()
            tokens[b, n] = rs.choice(V, p=w / w.sum())
    u = torch.rand(B, N, generator=gen)
    return tokens, parents, p, u, (q if dense else None)


def _same_walk(spec, tokens, parents, p, u, q, view=lambda x: x.cuda()):
    want = oracle.verify_tree(tokens, parents, p.numpy(), u.numpy(), None if q is None else q.numpy())
    got = spec.verify_tree(torch.from_numpy(tokens).cuda(), torch.from_numpy(parents).cuda(),
                           view(p), u.cuda(), None if q is None else view(q))
    for a, b in zip(got, want):
        assert np.array_equal(a.cpu().numpy(), b), (a, b)
    return want


@pytest.mark.parametrize("dense", [True, False])
@pytest.mark.parametrize("B,N,V", [
    (1, 1, 1), (3, 1, 7), (7, 2, 2), (64, 8, 3), (50, 12, 128), (40, 16, 129), (40, 33, 1000),
    (9, 64, 1024), (6, 24, 8192), (4, 20, 50257), (2, 12, 131072), (3, 256, 37), (1, 5, 200001),
])
def test_verify_matches_oracle(spec, B, N, V, dense):
    _same_walk(spec, *_verify_case(B, N, V, 100 * N + V, dense, ragged=N > 8))


def test_verify_walks_chains_and_many_siblings(spec):
    for fan, N in ((1, 40), (200, 200)):
        c = _verify_case(12, N, 50, 9, True, fan=fan)
        parents = np.arange(-1, N - 1) if fan == 1 else np.array([-1] + [0] * (N - 1))
        want = _same_walk(spec, c[0], np.tile(parents.astype(np.int32), (12, 1)), *c[2:])
        if fan == 1:
            assert want[1].max() > 3  # some walks go deep


def test_verify_accepts_everything_when_the_draft_is_the_target(spec):
    tokens, _, p, u, _ = _verify_case(16, 10, 300, 4, True)
    chain = np.tile(np.arange(-1, 9, dtype=np.int32), (16, 1))
    for b in range(16):
        for n in range(1, 10):
            tokens[b, n] = np.random.RandomState(b * 10 + n).choice(300, p=(lambda w: w / w.sum())(
                p[b, n - 1].double().numpy()))
    want = _same_walk(spec, tokens, chain, p, u, p)
    assert (want[1] == 10).all()


def test_verify_edges(spec):
    """Degenerate rows: nothing left of p, no weight at all, unknown tokens, u at its ends, NaN in
    rows that the walk does not visit, node 0 not a root."""
    V, N = 6, 4
    par = np.array([[-1, 0, 0, 1]], np.int32)
    one = torch.eye(V)
    u = torch.full((1, N), 0.999999)
    flat = torch.full((1, N, V), 1.0 / V)
    # p = q with a rejected child: nothing is left, the token comes from p again.
    q = flat.clone()
    p = flat.clone()
    p[0, 0] = torch.tensor([0.0, 0.2, 0.2, 0.2, 0.2, 0.2])
    q[0, 0] = torch.tensor([0.0, 0.2, 0.2, 0.2, 0.2, 0.2])
    _same_walk(spec, np.array([[0, 0, 0, 0]]), par, p, u, q)
    # No token has any weight.
    want = _same_walk(spec, np.array([[0, 1, 2, 3]]), par, torch.zeros(1, N, V), u, None)
    assert want[2][0] == -1 and want[1][0] == 1
    # Unknown tokens are never accepted; the last of u draws the last token.
    want = _same_walk(spec, np.array([[0, -1, V, 1 << 40]]), par, flat, u, None)
    assert want[1][0] == 1 and want[2][0] == V - 1
    want = _same_walk(spec, np.array([[0, -1, V, 1 << 40]]), par, flat, u * 0, flat)
    # One-hot target: greedy verification.
    greedy = one[torch.tensor([[3, 5, 1, 2]])]
    want = _same_walk(spec, np.array([[0, 2, 3, 1]]), par, greedy, u, None)
    assert want[0].tolist() == [[0, 2, -1, -1]] and want[2][0] == 1
    # u = 0 accepts any token of positive probability, and draws the first.
    want = _same_walk(spec, np.array([[0, 4, 3, 1]]), par, flat, u * 0, None)
    assert want[0].tolist() == [[0, 1, 3, -1]] and want[2][0] == 0
    # NaN in rows off the path.
    bad = flat.clone()
    bad[0, 2:] = float("nan")
    _same_walk(spec, np.array([[0, 4, 3, 1]]), np.array([[-1, 0, 0, 0]], np.int32), bad, u * 0, bad)
    # Node 0 not a root.
    want = _same_walk(spec, np.array([[0, 4, 3, 1]]), np.array([[-2, 0, 0, 1]], np.int32), flat, u, None)
    assert want[1][0] == 0 and want[2][0] == -1


@pytest.mark.parametrize("kind", ["padded", "node_slice", "offset", "feature"])
def test_verify_layouts(spec, kind):
    B, N, V = 5, 9, 260
    tokens, parents, p, u, q = _verify_case(B, N, V, 77, True)

    def view(x):
        x = x.cuda()
        if kind == "padded":      # rows of a padded vocabulary
            big = torch.full((B, N, V + 3), float("nan"), device="cuda")
            big[..., :V] = x
            return big[..., :V]
        if kind == "node_slice":
            big = torch.full((N, B, V), float("nan"), device="cuda")
            big.copy_(x.transpose(0, 1))
            return big.transpose(0, 1)
        if kind == "offset":
            flat = torch.zeros(x.numel() + 1, device="cuda")
            flat[1:] = x.flatten()
            return flat[1:].view(x.shape)
        return x.transpose(1, 2).contiguous().transpose(1, 2)

    _same_walk(spec, tokens, parents, p, u, q, view)


@pytest.mark.parametrize("dense", [True, False])
def test_verified_tokens_follow_the_target(spec, dense):
    """The token after the root, accepted or drawn, is distributed as the target's row 0: 2^18
    walks with two tries each. Pearson's statistic with V - 1 = 7 degrees of freedom stays below 45
    (probability above it 1.4e-7) for drawn children; for chosen ones too."""
    B, V = 1 << 18, 8
    gen = torch.Generator("cuda").manual_seed(5)
    p = torch.tensor([0.05, 0.3, 0.02, 0.13, 0.2, 0.1, 0.15, 0.05], device="cuda")
    q = torch.tensor([0.3, 0.1, 0.1, 0.1, 0.1, 0.1, 0.1, 0.1], device="cuda")
    tokens = torch.zeros(B, 3, dtype=torch.long, device="cuda")
    if dense:
        tokens[:, 1:] = torch.multinomial(q, 2 * B, replacement=True, generator=gen).view(B, 2)
    else:
        tokens[:, 1:] = torch.tensor([1, 6], device="cuda")
    u = torch.rand(B, 3, generator=gen, device="cuda")
    rows = p.expand(B, 3, V)
    path, counts, nxt = spec.verify_tree(tokens, torch.tensor([-1, 0, 0], device="cuda"), rows, u,
                                         q.expand(B, 3, V) if dense else None)
    first = torch.where(counts > 1, tokens.gather(1, path[:, 1:2].clamp(min=0).long())[:, 0], nxt)
    seen = torch.bincount(first, minlength=V).double()
    want = p.double() / p.double().sum() * B
    assert ((seen - want) ** 2 / want).sum().item() < 45
    assert 0.2 < (counts > 1).double().mean().item() < 0.99


@pytest.mark.parametrize("change,match", [
    (lambda a: a.update(target_probs=a["target_probs"].half()), "float32"),
    (lambda a: a.update(target_probs=a["target_probs"].cpu()), "CUDA"),
    (lambda a: a.update(target_probs=a["target_probs"][0]), "float32"),
    (lambda a: a.update(tokens=a["tokens"][:, :2]), "tokens"),
    (lambda a: a.update(tokens=a["tokens"].float()), "tokens"),
    (lambda a: a.update(tokens=a["tokens"].cpu()), "CUDA"),
    (lambda a: a.update(uniforms=a["uniforms"].double()), "uniforms"),
    (lambda a: a.update(uniforms=a["uniforms"][:1]), "uniforms"),
    (lambda a: a.update(parents=a["parents"][:, :2]), "parents"),
    (lambda a: a.update(draft_probs=a["draft_probs"][..., :4]), "draft_probs"),
    (lambda a: a.update(draft_probs=a["draft_probs"].double()), "draft_probs"),
])
def test_verify_refusals(spec, change, match):
    tokens, parents, p, u, q = _verify_case(2, 3, 5, 1, True)
    a = dict(tokens=torch.from_numpy(tokens).cuda(), parents=torch.from_numpy(parents).cuda(),
             target_probs=p.cuda(), uniforms=u.cuda(), draft_probs=q.cuda())
    change(a)
    with pytest.raises(RuntimeError, match=match):
        spec.verify_tree(**a)


# ------------------------------------------------------------------------------ commit

def _status():
    import ctypes
    from tiny_transformer_b200.operators._extension import load_c_abi
    flags = ctypes.c_uint(0)
    return load_c_abi().tt_attn_device_status(ctypes.byref(flags), 1), flags.value


@pytest.mark.parametrize("L,B,H,N,C,P", [(1, 1, 1, 1, 1, 1), (2, 3, 4, 9, 40, 9), (8, 5, 2, 16, 33, 5),
                                         (67, 2, 1, 4, 12, 4), (1, 300, 3, 6, 10, 6)])
def test_commit_matches_indexing(spec, L, B, H, N, C, P):
    gen, rs = torch.Generator().manual_seed(L + B), np.random.RandomState(L + B)
    ck = [_randn(gen, B, H, C, 64).cuda() for _ in range(L)]
    cv = [_randn(gen, B, H, C, 64).cuda() for _ in range(L)]
    kv = [_randn(gen, B, N, 2, H, 64).cuda() for _ in range(L)]
    tk, tv = ([x[:, :, i].transpose(1, 2) for x in kv] for i in range(2))
    counts = rs.randint(0, min(P, C) + 1, B)
    lens = np.array([rs.randint(0, C - c + 1) for c in counts])
    path = np.full((B, P), -1)
    for b in range(B):
        path[b, :counts[b]] = rs.randint(0, N, counts[b])
    want_k, want_v = [x.clone() for x in ck], [x.clone() for x in cv]
    for b in range(B):
        for i in range(counts[b]):
            for l in range(L):
                want_k[l][b, :, lens[b] + i] = tk[l][b, :, path[b, i]]
                want_v[l][b, :, lens[b] + i] = tv[l][b, :, path[b, i]]
    new = spec.commit_path(ck, cv, tk, tv, torch.from_numpy(path).cuda(),
                           torch.from_numpy(counts).cuda(), torch.from_numpy(lens).cuda())
    assert new.dtype == torch.int32 and new.tolist() == (lens + counts).tolist()
    for got, want in zip(ck + cv, want_k + want_v):
        assert torch.equal(got, want)
    assert _status() == (0, 0)


def test_commit_skips_what_does_not_fit(spec):
    B, H, N, C = 5, 2, 6, 10
    gen = torch.Generator().manual_seed(3)
    ck, cv = _randn(gen, B, H, C, 64).cuda(), _randn(gen, B, H, C, 64).cuda()
    tk, tv = _randn(gen, B, H, N, 64).cuda(), _randn(gen, B, H, N, 64).cuda()
    path = torch.tensor([[0, 1, 2], [3, 4, 5], [0, 7, -5], [1, 1, 1], [0, 2, 4]]).cuda()
    counts = torch.tensor([3, 3, 3, 2, 9]).cuda()     # the last one is more than the path holds
    lens = torch.tensor([8, 10, 0, -4, 4]).cuda()
    want_k, want_v = ck.clone(), cv.clone()
    for b, i, row, node in [(0, 0, 8, 0), (0, 1, 9, 1), (2, 0, 0, 0), (4, 0, 4, 0), (4, 1, 5, 2),
                            (4, 2, 6, 4)]:
        want_k[b, :, row], want_v[b, :, row] = tk[b, :, node], tv[b, :, node]
    assert _status() == (0, 0)
    new = spec.commit_path(ck, cv, tk, tv, path, counts, lens)
    assert new.tolist() == [10, 10, 3, -4, 7]
    assert torch.equal(ck, want_k) and torch.equal(cv, want_v)
    assert _status() == (1, 2) and _status() == (0, 0)


def test_commit_into_strided_caches_and_from_copied_trees(spec):
    """Token-major caches are written in place; trees that cannot be read in place are copied."""
    B, H, N, C = 2, 3, 4, 20
    gen = torch.Generator().manual_seed(8)
    store = _randn(gen, B, C, 2, H, 64).cuda()
    ck, cv = store[:, :, 0].transpose(1, 2), store[:, :, 1].transpose(1, 2)
    tree = _randn(gen, 2, B, H, 64, N).cuda().transpose(3, 4)
    path, counts = torch.tensor([[0, 2], [1, 3]]).cuda(), torch.tensor([2, 2]).cuda()
    lens = torch.tensor([0, 18]).cuda()
    spec.commit_path(ck, cv, tree[0], tree[1], path, counts, lens)
    assert torch.equal(ck[0, :, :2], tree[0][0][:, [0, 2]])
    assert torch.equal(cv[1, :, 18:], tree[1][1][:, [1, 3]])


@pytest.mark.parametrize("change,error,match", [
    (lambda a: a.update(cache_k=[]), RuntimeError, "layers"),
    (lambda a: a.update(tree_v=a["tree_v"] * 2), RuntimeError, "layers"),
    (lambda a: a.update(cache_k=[a["cache_k"][0].float()]), RuntimeError, "bf16"),
    (lambda a: a.update(cache_k=[a["cache_k"][0].cpu()]), RuntimeError, "CUDA"),
    (lambda a: a.update(cache_k=[a["cache_k"][0][..., ::2]]), RuntimeError, "head_dim=64"),
    (lambda a: a.update(cache_k=[a["cache_k"][0][:, :, :9]]), RuntimeError, "same shape"),
    (lambda a: a.update(cache_k=[a["cache_k"][0].transpose(2, 3).contiguous().transpose(2, 3)]),
     RuntimeError, "in place"),
    (lambda a: a.update(tree_k=[a["tree_k"][0][:, :1]]), RuntimeError, "trees must"),
    (lambda a: a.update(path=a["path"][:1]), RuntimeError, "path"),
    (lambda a: a.update(counts=a["counts"][:1]), RuntimeError, "counts"),
    (lambda a: a.update(counts=a["counts"].float()), RuntimeError, "int32 or int64"),
    (lambda a: a.update(cache_k=[a["cache_k"][0].requires_grad_()]), NotImplementedError, "backward"),
])
def test_commit_refusals(spec, change, error, match):
    x = lambda n: [torch.zeros(2, 2, n, 64, dtype=torch.bfloat16, device="cuda")]  # noqa: E731
    a = dict(cache_k=x(10), cache_v=x(10), tree_k=x(4), tree_v=x(4),
             path=torch.zeros(2, 3, dtype=torch.int32, device="cuda"),
             counts=torch.ones(2, dtype=torch.int32, device="cuda"),
             cache_lens=torch.zeros(2, dtype=torch.int32, device="cuda"))
    change(a)
    with pytest.raises(error, match=match):
        spec.commit_path(**a)


@pytest.mark.parametrize("N", [4, 40])
def test_back_to_back_calls_see_each_other(spec, N):
    """Programmatic launches overlap a kernel's start with the end of the one before it: a chain in
    which every call reads what the last one wrote gives the same with and without waiting between
    the calls. (4 nodes: the cluster kernel; 40: the persistent one.)"""
    B, H, C, V = 3, 2, 600, 1000
    gen = torch.Generator().manual_seed(17)
    q, tk, tv = (_randn(gen, B, H, N, 64).cuda() for _ in range(3))
    parents = torch.arange(-1, N - 1, dtype=torch.int32).cuda()
    p = torch.softmax(torch.randn(B, N, V, generator=gen) * 3, -1).cuda()
    uniforms = torch.rand(60, B, N, generator=gen).cuda()
    start = [_randn(gen, B, H, C, 64).cuda() for _ in range(2)]

    def chain(wait):
        ck, cv = (x.clone() for x in start)
        lens = torch.zeros(B, dtype=torch.int32, device="cuda")
        tokens = torch.zeros(B, N, dtype=torch.long, device="cuda")
        k, v, seen = tk.clone(), tv.clone(), []
        for step in range(60):
            o = spec.tree_attention(q, k, v, ck, cv, parents, lens)
            if wait:
                torch.cuda.synchronize()
            path, counts, nxt = spec.verify_tree(tokens, parents, p, uniforms[step], p)
            if wait:
                torch.cuda.synchronize()
            counts = counts.clamp(max=9)
            lens = spec.commit_path(ck, cv, k, v, path, counts, lens)
            if wait:
                torch.cuda.synchronize()
            k, v = o, o * 0.5 + v * 0.5           # the next step's rows come from this one's output
            tokens = (tokens + nxt[:, None]) % V
            seen.append(nxt)
        return o, lens, ck, cv, torch.stack(seen)

    want = chain(True)
    for _ in range(5):
        for a, b in zip(chain(False), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dense", [True, False])
@pytest.mark.parametrize("B,V", [(1, 1 << 22), (99, 920001), (150, 460001)])
def test_verify_largest_shares_of_the_vocabulary(spec, B, V, dense):
    """The most windows a CTA takes: the largest vocabulary, and large ones on as few CTAs a sequence as
    the batch leaves (2 and 1). One row of probabilities for the whole batch, other draws."""
    rs = np.random.RandomState(V % 1000)
    gen = torch.Generator().manual_seed(V)
    logits = torch.randn(1, 2, V, generator=gen) * 2
    p = torch.softmax(logits, -1)
    q = torch.softmax(logits + torch.randn(1, 2, V, generator=gen), -1)
    w = q[0, 0].double().numpy()
    tokens = np.zeros((B, 2), np.int64)
    tokens[:, 1] = rs.choice(V, B, p=w / w.sum())
    u = torch.rand(B, 2, generator=gen)
    want = _same_walk(spec, tokens, np.tile(np.array([[-1, 0]], np.int32), (B, 1)), p.expand(B, 2, V), u,
                      q.expand(B, 2, V) if dense else None,
                      lambda x: x[:1].cuda().expand(B, 2, V))
    assert (want[2] >= 0).all()


# ------------------------------------------------------------------------------ errors of launches

class _LegacyStreamClosed:
    """While a blocking stream is being captured, a launch into the legacy stream is refused by the
    driver (and ends the capture as invalid): a launch failure that nothing of it reaches the GPU."""

    def __enter__(self):
        import ctypes
        self.cuda, self.stream = ctypes.CDLL("libcuda.so.1"), ctypes.c_void_p()
        assert self.cuda.cuStreamCreate(ctypes.byref(self.stream), 0) == 0
        assert self.cuda.cuStreamBeginCapture_v2(self.stream, 0) == 0

    def __exit__(self, *_):
        import ctypes
        graph = ctypes.c_void_p()
        self.cuda.cuStreamEndCapture(self.stream, ctypes.byref(graph))
        assert not graph.value
        assert self.cuda.cuStreamDestroy_v2(self.stream) == 0


@pytest.mark.parametrize("failing", ["tree", "large tree", "verify", "commit", "decode"])
def test_a_failed_launch_is_reported_once(failing):
    """By the call that failed, and not again by the next one."""
    import ctypes
    from tiny_transformer_b200.operators._extension import load_c_abi
    lib = load_c_abi()
    B, H, C, V = 1, 1, 64, 10
    make = lambda n: torch.zeros(B, H, n, 64, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    cache, rows, out, query = make(C), make(40), make(40), make(1)
    ints = torch.zeros(2, 40, dtype=torch.int32, device="cuda")
    parents = torch.arange(-1, 39, dtype=torch.int32, device="cuda")
    tokens, drawn = (torch.zeros(B, 40, dtype=torch.long, device="cuda") for _ in range(2))
    probs = torch.full((B, 40, V), 1 / V, device="cuda")
    u, lse = torch.zeros(B, 40, device="cuda"), torch.zeros(B, H, 40, device="cuda")
    work = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    s = lambda x: (ctypes.c_int64 * 4)(*x.stride())  # noqa: E731
    one = lambda x: (ctypes.c_void_p * 1)(x.data_ptr())  # noqa: E731
    assert lib.tt_attn_tree_workspace_size(B, H, H, 40, C) <= work.numel()

    def tree(nodes):
        return lib.tt_attn_tree_forward_bf16(
            rows.data_ptr(), s(rows), rows.data_ptr(), s(rows), rows.data_ptr(), s(rows),
            cache.data_ptr(), s(cache), cache.data_ptr(), s(cache), B, H, H, nodes, C, 64,
            parents.data_ptr(), 0, None, out.data_ptr(), None, work.data_ptr(), work.numel(), None)

    calls = {
        "tree": lambda: tree(4),
        "large tree": lambda: tree(40),
        "verify": lambda: lib.tt_attn_tree_verify_f32(
            tokens.data_ptr(), parents.data_ptr(), 0, probs.data_ptr(), 40 * V, V, None, 0, 0,
            u.data_ptr(), B, 40, V, ints.data_ptr(), ints[1].data_ptr(), drawn.data_ptr(), None),
        "commit": lambda: lib.tt_attn_tree_commit_bf16(
            one(cache), s(cache), one(cache), s(cache), one(rows), s(rows), one(rows), s(rows), 1, B,
            H, 40, C, 64, ints.data_ptr(), 40, ints[1].data_ptr(), ints[1, 1:].data_ptr(),
            ints[1, 2:].data_ptr(), None),
        "decode": lambda: lib.tt_attn_forward_bf16(
            query.data_ptr(), s(query), cache.data_ptr(), s(cache), cache.data_ptr(), s(cache), B, H, 1,
            C, 64, C - 1, None, out.data_ptr(), lse.data_ptr(), None, 0, None),
    }
    assert lib.tt_attn_forward_workspace_size(B, H, 1, C) == 0
    for name, call in calls.items():
        assert call() == 0, (name, lib.tt_attn_last_error())
    torch.cuda.synchronize()
    with _LegacyStreamClosed():
        status = calls[failing]()
    assert status != 0 and "launch" in lib.tt_attn_last_error().decode()
    for name, call in calls.items():
        assert call() == 0, (name, lib.tt_attn_last_error())
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------ long caches, value by value

def marked_values(rows):
    """V rows of which each has one entry, 1, at a place that differs within every 64 rows and from one
    64 rows to the next: a V row that is lost, doubled or out of its place moves weight between features.
    No entry is negative, so A equals |ref| and the bound of the file is relative: 2^-7 + 2^-11."""
    j = torch.arange(rows)
    return torch.nn.functional.one_hot((j + 7 * (j // 64)) % 64, 64).to(torch.bfloat16)


@pytest.mark.parametrize("Hq,Hkv,N,C,lens", [
    (2, 2, 3, 9000, [8999, 4097]),      # the cluster kernel, cache shared by its CTAs
    (3, 1, 8, 9000, [9000, 2500]),      # the same, two row tiles
    (2, 2, 40, 9000, [8999, 4097]),     # the persistent kernel: two copies of Q
    (1, 1, 33, 20001, [20001, 64]),     # one long unit shared by many CTAs
    (3, 1, 37, 9000, [9000, 129]),      # 111 rows: one copy
    (2, 1, 130, 6000, [5999, 3000]),    # 260 rows in three tiles, two key tiles of the tree
])
def test_every_value_of_a_long_cache_has_its_weight(spec, Hq, Hkv, N, C, lens):
    B = len(lens)
    t, parents, _ = _case(B, Hq, Hkv, N, C, 17 * N + C)
    t["cache_v"] = marked_values(C).expand(B, Hkv, C, 64).contiguous()
    t["tree_v"] = marked_values(N).expand(B, Hkv, N, 64).contiguous()
    o, lse = _run(spec, t, parents, lens)
    _check(o, lse, t, parents, lens)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("G,N", [(1, 12), (1, 30), (3, 16), (2, 64)])
def test_a_leaf_that_is_not_finite_shows_in_its_own_row(spec, value, G, N):
    """K and V of one leaf: every feature of that node's row, in every head, and no other row."""
    lens = [130, 0]
    t, parents, _ = _case(2, 2 * G, 2, N, 300, 11, fan=4)
    want, want_lse = _run(spec, t, parents, lens)
    leaf = [n for n in range(N) if n not in parents[0]][-1]
    t["tree_k"][0, :, leaf] = value
    t["tree_v"][0, :, leaf] = value
    got, lse = _run(spec, t, parents, lens)
    assert not torch.isfinite(got[0, :, leaf]).any() and not torch.isfinite(lse[0, :, leaf]).any()
    others = [n for n in range(N) if n != leaf]
    assert torch.equal(got[0][:, others], want[0][:, others]) and torch.equal(got[1], want[1])
    assert torch.equal(lse[0][:, others], want_lse[0][:, others]) and torch.equal(lse[1], want_lse[1])
