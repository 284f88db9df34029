"""Query/key norm with the rotation on the GPU, forward and backward, against its 64-bit restatement.

Tolerances. Forward: at most 8 FP32 roundings and a reciprocal root, together below 2^-20 of the magnitudes of an
element's two terms, then bf16 (2^-8 of the result). dx: its terms have a magnitude bound M (oracle); the rotation, the two
sums of 64 and the products take fewer than 24 roundings, each within 2^-24 of a term: 2^-18 M covers them (24 * 2^-24 and the
root's 2^-21), then bf16. dw: a thread adds at most N of its rows in FP32, 16 threads' sums after that, then
64 bits: (N + 16) 2^-24 of the sum of magnitudes; N is below 256 for the sizes here, so 2^-15, then the type's
rounding.
"""
import ctypes

import numpy as np
import pytest
import torch

from oracle import cache4_oracle as oracle

pytestmark = pytest.mark.gpu

EPS = 1e-6


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available() or torch.cuda.get_device_capability()[0] != 10:
        pytest.skip("needs an sm_100 GPU")


@pytest.fixture(scope="module")
def op():
    from tiny_transformer_b200.operators import fused
    return fused.qkv_norm_rope


def _status():
    from tiny_transformer_b200.operators._extension import load_c_abi
    flags = ctypes.c_uint(0)
    load_c_abi().tt_attn_device_status(ctypes.byref(flags), 1)
    return flags.value


def _tables(n=400):
    angle = torch.arange(n).double()[:, None] / 10000 ** (torch.arange(0, 64, 2).double() / 64)
    return angle.cos().float(), angle.sin().float()


def _inputs(B, T, Hq, Hkv, weights, seed):
    gen = torch.Generator().manual_seed(seed)
    heads = Hq + 2 * Hkv
    qkv = (torch.randn(B, T, heads, 64, generator=gen) *
           torch.exp(0.7 * torch.randn(heads, 64, generator=gen))).to(torch.bfloat16)
    w = [None, None]
    if weights is not None:
        w = [(1 + 0.3 * torch.randn(64, generator=gen)).to(weights) for _ in range(2)]
    g = [torch.randn(B, h, T, 64, generator=gen).to(torch.bfloat16) for h in (Hq, Hkv, Hkv)]
    return qkv, w, g


def _np(x):
    return None if x is None else x.detach().double().cpu().numpy()


def _positions(kind, B, T):
    """The argument and the [B, T] positions it stands for."""
    if kind == "each":
        first = torch.tensor([(17 * b + 3) % 100 for b in range(B)])
        return first.cuda(), (first[:, None] + torch.arange(T)).numpy()
    if kind == "one":
        return torch.tensor([9], device="cuda"), np.broadcast_to(9 + np.arange(T), (B, T))
    if kind == "every":
        at = torch.randint(0, 400, (B, T), generator=torch.Generator().manual_seed(T))
        return at.cuda(), at.numpy()
    return kind, np.broadcast_to(kind + np.arange(T), (B, T))


def _expected(qkv, w, g, at, Hq, Hkv):
    cos, sin = (_np(t)[at] for t in _tables())
    x = _np(qkv)
    out, dx, bound, dw, dwb = [], [], [], [], []
    for i, part in enumerate((x[:, :, :Hq], x[:, :, Hq:Hq + Hkv])):
        y, mag = oracle.norm_rope(part, _np(w[i]), cos, sin, EPS)
        out.append((y.transpose(0, 2, 1, 3), mag.transpose(0, 2, 1, 3)))
        d, dwi, m, mw = oracle.norm_rope_backward(part, _np(w[i]), cos, sin, EPS, _np(g[i]).transpose(0, 2, 1, 3))
        dx.append(d)
        bound.append(m)
        dw.append(dwi)
        dwb.append(mw)
    dx.append(_np(g[2]).transpose(0, 2, 1, 3))
    bound.append(np.zeros_like(dx[2]))
    return out, np.concatenate(dx, 2), np.concatenate(bound, 2), dw, dwb


def _check(got, grads, want, w):
    out, dx, bound, dw, dwb = want
    for y, (ref, mag) in zip(got, out):
        assert y.is_contiguous()
        assert (np.abs(_np(y) - ref) <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -20 * mag).all()
    assert (np.abs(_np(grads[0]).reshape(dx.shape) - dx) <= 2.0 ** -8 * np.abs(dx) + 2.0 ** -18 * bound).all()
    for i in range(2):
        if w[i] is not None:
            assert grads[1 + i].dtype == w[i].dtype
            err = np.abs(_np(grads[1 + i]) - dw[i])
            assert (err <= torch.finfo(w[i].dtype).eps / 2 * np.abs(dw[i]) + 2.0 ** -15 * dwb[i]).all(), err.max()


@pytest.mark.parametrize("B,T,Hq,Hkv,weights,position", [
    (1, 1, 1, 1, torch.bfloat16, 0),
    (1, 1, 12, 12, torch.float32, 399),
    (2, 5, 12, 12, torch.bfloat16, 7),
    (3, 33, 6, 2, torch.float32, "each"),
    (2, 130, 9, 1, torch.bfloat16, "one"),
    (3, 127, 4, 4, torch.bfloat16, "every"),
    (2, 64, 8, 2, None, 100),
    (5, 3, 2, 1, None, "every"),
    (4, 300, 12, 4, torch.float32, "each"),
])
def test_matches_oracle(op, B, T, Hq, Hkv, weights, position):
    qkv, w, g = _inputs(B, T, Hq, Hkv, weights, 31 * T + Hq)
    arg, at = _positions(position, B, T)
    cos, sin = (t.cuda() for t in _tables())
    leaves = [x.cuda().requires_grad_() for x in (qkv, *w) if x is not None]
    args = leaves if weights is not None else [leaves[0], None, None]
    q, k, v = op(*args, cos, sin, arg, EPS, Hkv)
    assert torch.equal(v.cpu(), qkv[:, :, Hq + Hkv:].transpose(1, 2)) and v.data_ptr() != q.data_ptr()
    grads = torch.autograd.grad((q, k, v), leaves, [x.cuda() for x in g], retain_graph=True)
    _check((q, k), grads, _expected(qkv, w, g, at, Hq, Hkv), w)
    # The same bits without a graph, and on a second backward.
    with torch.no_grad():
        q2, k2, v2 = op(*args, cos, sin, arg, EPS, Hkv)
    assert torch.equal(q, q2) and torch.equal(k, k2) and v2.data_ptr() == args[0][:, :, Hq + Hkv:].data_ptr()
    again = torch.autograd.grad((q, k, v), leaves, [x.cuda() for x in g])
    assert all(map(torch.equal, grads, again))
    assert _status() == 0


def test_gradient_against_differences(op):
    """The loss' change along a direction, in 64 bits from the forward's formula at bf16 inputs."""
    B, T, H = 1, 6, 2
    qkv, w, g = _inputs(B, T, H, H, torch.float32, 5)
    cos, sin = _tables()
    at = np.broadcast_to(np.arange(T), (B, T))
    c, s = _np(cos)[at], _np(sin)[at]

    def loss(x, wq, wk):
        q, _ = oracle.norm_rope(x[:, :, :H], wq, c, s, EPS)
        k, _ = oracle.norm_rope(x[:, :, H:2 * H], wk, c, s, EPS)
        return sum((y.transpose(0, 2, 1, 3) * _np(gi)).sum() for y, gi in zip((q, k, x[:, :, 2 * H:]), g))

    leaves = [x.cuda().requires_grad_() for x in (qkv, *w)]
    out = op(*leaves, cos.cuda(), sin.cuda(), 0, EPS, H)
    grads = torch.autograd.grad(out, leaves, [x.cuda() for x in g])
    rs = np.random.RandomState(1)
    for i, x in enumerate((qkv, *w)):
        d = rs.randn(*x.shape)
        base = [_np(t) for t in (qkv, *w)]
        h = 1e-5
        plus = [b + h * d if j == i else b for j, b in enumerate(base)]
        minus = [b - h * d if j == i else b for j, b in enumerate(base)]
        diff = (loss(*plus) - loss(*minus)) / (2 * h)
        size = (np.abs(_np(grads[i])) * np.abs(d)).sum()
        assert abs((_np(grads[i]) * d).sum() - diff) <= 2.0 ** -8 * size + 1e-4


def test_layouts_and_missing_gradients(op):
    B, T, H = 2, 11, 3
    qkv, w, g = _inputs(B, T, H, H, torch.bfloat16, 9)
    cos, sin = (t.cuda() for t in _tables())
    w = [x.cuda().requires_grad_() for x in w]
    base = qkv.cuda()
    g = [x.cuda() for x in g]

    def run(x, g, which=(0, 1, 2)):
        x = x.detach().requires_grad_()
        out = op(x, *w, cos, sin, 4, EPS, None if x.dim() == 5 else H)
        grads = torch.autograd.grad([out[i] for i in which], [x, *w], [g[i] for i in which], allow_unused=True)
        return out, grads

    want, wgrads = run(base, g)
    wide = torch.zeros(B, T + 2, 3 * H + 2, 64, dtype=torch.bfloat16, device="cuda")
    wide[:, 2:, 1:-1] = base
    odd = torch.zeros(base.numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view_as(base).copy_(base)
    token_major = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in g]
    spread = [torch.zeros(*x.shape[:3], 128, dtype=x.dtype, device="cuda")[..., ::2].copy_(x) for x in g]
    for x, gg in ((base.view(B, T, 3, H, 64), g), (wide[:, 2:, 1:-1], token_major), (odd, spread)):
        out, grads = run(x, gg)
        assert all(map(torch.equal, want, out))
        assert all(torch.equal(a, b.view_as(a)) for a, b in zip(wgrads, grads))
    zero = [torch.zeros_like(x) for x in g]
    for which in ((0,), (1,), (2,), (0, 2)):
        _, grads = run(base, g, which)
        _, full = run(base, [g[i] if i in which else zero[i] for i in range(3)])
        assert all(map(torch.equal, full, grads))
    # Expanded gradients (a sum's) and only some leaves.
    x = base.clone().requires_grad_()
    q, k, v = op(x, *w, cos, sin, 4, EPS, H)
    (q.float().sum() + k.float().sum() + v.float().sum()).backward()
    ones, full = run(base, [torch.ones_like(t) for t in g])
    assert torch.equal(x.grad, full[0]) and torch.equal(w[0].grad, full[1]) and torch.equal(w[1].grad, full[2])
    q, k, _ = op(base, *w, cos, sin, 4, EPS, H)
    only = torch.autograd.grad((q, k), w, g[:2])
    assert torch.equal(only[0], wgrads[1]) and torch.equal(only[1], wgrads[2])


def test_in_front_of_the_attention(op):
    """The whole of a block's attention, trained: gradients of the projection through student.attention."""
    from tiny_transformer_b200.operators import student
    B, T, H = 2, 150, 2
    qkv, w, _ = _inputs(B, T, H, H, torch.bfloat16, 12)
    cos, sin = (t.cuda() for t in _tables())
    do = torch.randn(B, H, T, 64, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    leaves = [x.cuda().requires_grad_() for x in (qkv, *w)]
    q, k, v = op(*leaves, cos, sin, 0, EPS, H)
    o = student.attention(q, k, v)
    got = torch.autograd.grad(o, leaves, do)
    ref = [x.detach().double().requires_grad_() for x in leaves]
    c, s = cos[:T].double()[None, :, None], sin[:T].double()[None, :, None]

    def turn(x, weight):
        n = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight
        e, o = n[..., 0::2], n[..., 1::2]
        return torch.stack((e * c - o * s, e * s + o * c), -1).flatten(-2).transpose(1, 2)

    qr, kr = turn(ref[0][:, :, :H], ref[1]), turn(ref[0][:, :, H:2 * H], ref[2])
    scores = qr @ kr.transpose(-1, -2) / 8
    scores = scores.masked_fill(~torch.ones(T, T, dtype=torch.bool, device="cuda").tril(), float("-inf"))
    want_o = torch.softmax(scores, -1) @ ref[0][:, :, 2 * H:].transpose(1, 2)
    want = torch.autograd.grad(want_o, ref, do.double())
    # bf16 throughout: q, k, P, dS, O and the gradients are each rounded (2^-8); six roundings of terms of the whole.
    assert (o.double() - want_o).norm() <= 6 * 2.0 ** -8 * want_o.norm()
    for a, b in zip(got, want):
        assert (a.double() - b).norm() <= 6 * 2.0 ** -8 * b.norm()


def test_rows_outside_the_table(op):
    B, T, H = 2, 3, 2
    qkv, w, g = _inputs(B, T, H, H, torch.bfloat16, 14)
    cos, sin = (t.cuda() for t in _tables(50))
    leaves = [x.cuda().requires_grad_() for x in (qkv, *w)]
    at = torch.tensor([[0, 50, 2], [-1, 7, 2**40]], device="cuda")
    inside = ((at >= 0) & (at < 50)).cpu()
    _status()
    q, k, v = op(*leaves, cos, sin, at, EPS, H)
    assert _status() == 2
    for y in (q, k):
        assert torch.equal((y != 0).any(-1).any(1).cpu(), inside)
    grads = torch.autograd.grad((q, k, v), leaves, [x.cuda() for x in g])
    assert _status() == 2
    assert torch.equal((grads[0][:, :, :2 * H] != 0).any(-1).any(-1).cpu(), inside)
    assert torch.equal(grads[0][:, :, 2 * H:], g[2].transpose(1, 2).cuda())
    assert grads[1].isfinite().all()
    for bad in (-1, 48):
        with pytest.raises(RuntimeError, match="table"):
            op(*leaves, cos, sin, bad, EPS, H)


def test_zero_rows_and_values_that_are_not_finite(op):
    qkv, w, g = _inputs(1, 4, 1, 1, torch.float32, 15)
    qkv[0, 0] = 0
    qkv[0, 1, 0, 5] = float("nan")
    cos, sin = (t.cuda() for t in _tables())
    leaves = [x.cuda().requires_grad_() for x in (qkv, *w)]
    q, k, v = op(*leaves, cos, sin, 0, EPS, 1)
    assert (q[0, 0, 0] == 0).all() and q[0, 0, 1].isnan().all() and q[0, 0, 2:].isfinite().all()
    dx, dqw, dkw = torch.autograd.grad((q, k, v), leaves, [x.cuda() for x in g])
    assert dx[0, 0].isfinite().all() and dx[0, 1, 0].isnan().all() and dx[0, 2:].isfinite().all()
    assert dqw.isnan().all() and dkw.isfinite().all()


def test_captured_training_step(op):
    B, T, H = 2, 40, 3
    cos, sin = (t.cuda() for t in _tables())
    qkv, w, g = _inputs(B, T, H, H, torch.bfloat16, 16)
    g = [x.cuda() for x in g]
    leaves = [x.cuda().requires_grad_() for x in (qkv, *w)]

    def step():
        return torch.autograd.grad(op(*leaves, cos, sin, 3, EPS, H), leaves, g)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (17, 18):
        new, _, _ = _inputs(B, T, H, H, torch.bfloat16, seed)
        with torch.no_grad():
            leaves[0].copy_(new)
        graph.replay()
        assert all(map(torch.equal, got, step()))


def test_capture_beside_an_eager_graph(op):
    """A living graph of the same leaves: from the default stream the capture is refused, from another one it works."""
    B, T, H = 1, 9, 2
    cos, sin = (t.cuda() for t in _tables())
    qkv, w, g = _inputs(B, T, H, H, torch.bfloat16, 19)
    g = [x.cuda() for x in g]
    leaves = [x.cuda().requires_grad_() for x in (qkv, *w)]

    def step():
        return torch.autograd.grad(op(*leaves, cos, sin, 3, EPS, H), leaves, g)

    held = op(*leaves, cos, sin, 3, EPS, H)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step()
    want = torch.autograd.grad(held, leaves, g)     # the eager graph is as it was
    del held
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        held = op(*leaves, cos, sin, 3, EPS, H)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for x in got:
        x.zero_()
    graph.replay()
    assert all(map(torch.equal, got, want))
    assert all(map(torch.equal, torch.autograd.grad(held, leaves, g), want))


@pytest.mark.parametrize("change,match", [
    (dict(qkv=lambda x: x.float()), "bf16"),
    (dict(qkv=lambda x: x[..., :32]), "head_dim=64"),
    (dict(kv_heads=lambda x: None), "kv_heads given"),
    (dict(kv_heads=lambda x: 3), "multiple"),
    (dict(kv_heads=lambda x: 0), "multiple"),
    (dict(cos=lambda x: x[:, ::2]), "tables"),
    (dict(sin=lambda x: x.cpu()), "same device"),
    (dict(position=lambda x: torch.zeros(2, 4, dtype=torch.long, device="cuda")), r"\[B, T\]"),
    (dict(q_weight=lambda x: None), "both norm weights"),
    (dict(q_weight=lambda x: x.half()), "bf16 or both be float32"),
    (dict(eps=lambda x: float("inf")), "eps"),
])
def test_refusals(op, change, match):
    qkv, w, _ = _inputs(2, 3, 4, 2, torch.bfloat16, 1)
    cos, sin = (t.cuda() for t in _tables())
    args = dict(qkv=qkv.cuda(), q_weight=w[0].cuda(), k_weight=w[1].cuda(), cos=cos, sin=sin, position=0, eps=EPS,
                kv_heads=2)
    for key, f in change.items():
        args[key] = f(args[key])
    with pytest.raises(RuntimeError, match=match):
        op(**args)
    args["qkv"] = args["qkv"].detach().requires_grad_()
    with pytest.raises(RuntimeError, match=match):
        op(**args)
    with pytest.raises(NotImplementedError, match="tables"):
        op(qkv.cuda(), *[x.cuda() for x in w], cos.requires_grad_(), sin, 0, EPS, 2)


def test_gradients_have_no_backward(op):
    qkv, w, g = _inputs(1, 4, 1, 1, torch.bfloat16, 1)
    cos, sin = (t.cuda() for t in _tables())
    leaves = [x.cuda().requires_grad_() for x in (qkv, *w)]
    want = torch.autograd.grad(op(*leaves, cos, sin, 0, EPS, 1), leaves, [x.cuda() for x in g])
    grads = torch.autograd.grad(op(*leaves, cos, sin, 0, EPS, 1), leaves, [x.cuda() for x in g], create_graph=True)
    assert all(map(torch.equal, want, grads))
    with pytest.raises(RuntimeError, match="no backward"):
        grads[0].sum().backward()
    # A projection changed between forward and backward is noticed.
    x = leaves[0].detach().clone().requires_grad_()
    y = x * 1
    out = op(y, *leaves[1:], cos, sin, 0, EPS, 1)
    with torch.no_grad():
        y.add_(1)
    with pytest.raises(RuntimeError, match="modified"):
        torch.autograd.grad(out, x, [t.cuda() for t in g])


def test_autocast_is_refused(op):
    qkv, w, _ = _inputs(1, 3, 1, 1, torch.bfloat16, 1)
    cos, sin = (t.cuda() for t in _tables())
    with torch.autocast("cuda", torch.bfloat16), pytest.raises(RuntimeError, match="AMP"):
        op(qkv.cuda(), *[x.cuda() for x in w], cos, sin, 0, EPS, 1)


@pytest.mark.parametrize("which", range(5))
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_derivatives_are_refused(op, which, grad):
    """A tangent would reach v, a view, and be lost from q and k."""
    import torch.autograd.forward_ad as forward_ad
    qkv, w, _ = _inputs(1, 3, 2, 2, torch.bfloat16, 1)
    inputs = [qkv.cuda(), *(x.cuda() for x in w), *(t.cuda() for t in _tables())]
    want = op(*inputs, 0, EPS, 2)
    if grad:
        inputs[0].requires_grad_()
    with forward_ad.dual_level():
        dual = list(inputs)
        dual[which] = forward_ad.make_dual(inputs[which], torch.ones_like(inputs[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            op(*dual, 0, EPS, 2)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            op(*dual, 0, EPS, 2)
        assert all(map(torch.equal, op(*inputs, 0, EPS, 2), want))
        plain = [forward_ad.unpack_dual(x).primal for x in dual]
        assert all(map(torch.equal, op(*plain, 0, EPS, 2), want))


def test_forward_mode_derivatives_of_the_gradients_are_refused(op):
    import torch.autograd.forward_ad as forward_ad
    qkv, w, g = _inputs(1, 3, 2, 2, torch.bfloat16, 1)
    cos, sin = (t.cuda() for t in _tables())
    leaves = [x.cuda().requires_grad_() for x in (qkv, *w)]
    g = [x.cuda() for x in g]
    out = op(*leaves, cos, sin, 0, EPS, 2)
    for i in range(2):
        with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(out[i], leaves, forward_ad.make_dual(g[i], g[i]), retain_graph=True, allow_unused=True)
    assert torch.autograd.grad(out, leaves, g)[0].isfinite().all()


def test_shared_heads_in_front_of_the_attention(op):
    """Shared K/V heads are repeated for student.attention, which wants as many K/V as query heads: values and gradients as
    from a projection that holds the repeated heads."""
    from tiny_transformer_b200.operators import student
    B, T, Hq, Hkv = 2, 70, 6, 2
    qkv, w, _ = _inputs(B, T, Hq, Hkv, torch.bfloat16, 31)
    cos, sin = (t.cuda() for t in _tables())
    do = torch.randn(B, Hq, T, 64, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    leaves = [x.cuda().requires_grad_() for x in (qkv, *w)]
    q, k, v = op(*leaves, cos, sin, 0, EPS, Hkv)
    with pytest.raises(RuntimeError, match="second dimension"):
        student.attention(q, k, v)
    k, v = (x.repeat_interleave(Hq // Hkv, 1) for x in (k, v))
    o = student.attention(q, k, v)
    got = torch.autograd.grad(o, leaves, do)
    wide = torch.cat([qkv[:, :, :Hq], *(x.repeat_interleave(Hq // Hkv, 2) for x in qkv[:, :, Hq:].split(Hkv, 2))], 2)
    wide = [x.cuda().requires_grad_() for x in (wide, *w)]
    want_o = student.attention(*op(*wide, cos, sin, 0, EPS, Hq))
    want = torch.autograd.grad(want_o, wide, do)
    assert torch.equal(o, want_o)
    k_v = want[0][:, :, Hq:].double().unflatten(2, (2 * Hkv, -1)).sum(3)
    dx = torch.cat([want[0][:, :, :Hq].double(), k_v], 2)
    # Both round the same sums of bf16 gradients once or twice more: three roundings of terms of the whole.
    for a, b in zip(got, (dx, *want[1:])):
        assert (a.double() - b.double()).norm() <= 3 * 2.0 ** -8 * b.double().norm()
