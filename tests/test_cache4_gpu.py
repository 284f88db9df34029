"""4-bit KV cache on the GPU against its 64-bit restatement (oracle/cache4_oracle.py).

Tolerances. Appended values: equal, code by code (the keys' bf16 values are rounded correctly; the oracle's are rounded
from 64 bits). q: FP32 arithmetic with at most 8 roundings and a root (2^-20 of the magnitudes of its two terms), then
bf16 (2^-8). Reading back: exact. Attention: K and V are exact in half precision; P is rounded to half precision (2^-11
of each weight); scores are FP32 sums of 64 products with sum |q k| / 8 below 32 for the inputs here, so off by 64 *
2^-23 * 32 = 2^-12 at most, which is 2^-11 in weight and normalisation together; the rest is below 2^-16. So
|O - ref| <= 2^-8 |ref| + 2^-9 A with A the same average of |v| (2^-11 + 2^-11 + 2^-16 < 2^-9). Half precision ends:
a weight is held as 2^7 times its ratio to the running maximum, which no weight of the row's end result is below by
definition of a maximum, and halves have steps of 2^-24, so a weight is also off by 2^-25 / 2^7 = 2^-32 of the largest
one, which is at most the sum: 2^-32 S more, S the sum of |v| over the rows. LSE: 2^-12 from the scores and 2^-20 of
its value from the logarithm.
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
def c4():
    from tiny_transformer_b200.operators import cache4
    return cache4


@pytest.fixture(scope="module")
def fused():
    from tiny_transformer_b200.operators import fused
    return fused


def _status(clear=True):
    from tiny_transformer_b200.operators._extension import load_c_abi
    flags = ctypes.c_uint(0)
    load_c_abi().tt_attn_device_status(ctypes.byref(flags), int(clear))
    return flags.value


def _tables(n):
    angle = torch.arange(n).double()[:, None] / 10000 ** (torch.arange(0, 64, 2).double() / 64)
    return angle.cos().float(), angle.sin().float()


def _projection(B, T, Hq, Hkv, seed, weights="bf16"):
    gen = torch.Generator().manual_seed(seed)
    heads = Hq + 2 * Hkv
    size = torch.exp(0.7 * torch.randn(heads, 64, generator=gen))
    qkv = (torch.randn(B, T, heads, 64, generator=gen) * size).to(torch.bfloat16)
    if weights is None:
        return qkv, None, None
    w = [1 + 0.3 * torch.randn(64, generator=gen) for _ in range(2)]
    if weights == "bf16":
        w = [x.to(torch.bfloat16) for x in w]
    return (qkv, *w)


def _np(x):
    return None if x is None else x.double().cpu().numpy()


def _reference(qkv, qw, kw, at, Hq, Hkv):
    """q (unrounded) and its terms' magnitudes, k rounded to bf16, v; [B, T, heads, 64]; at [B, T] positions."""
    cos, sin = (_np(t)[at] for t in _tables(at.max() + 1))
    x = _np(qkv)
    q, mag = oracle.norm_rope(x[:, :, :Hq], _np(qw), cos, sin, EPS)
    k, _ = oracle.norm_rope(x[:, :, Hq:Hq + Hkv], _np(kw), cos, sin, EPS)
    k = torch.from_numpy(k).to(torch.bfloat16).double().numpy()
    return q, mag, k, x[:, :, Hq + Hkv:]


def _check_q(q, ref, mag):
    q = _np(q).transpose(0, 2, 1, 3)
    assert (np.abs(q - ref) <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -20 * mag).all()


def _check_rows(cache, rows, at):
    """Rows [B, T, Hkv, 64] at positions [B, T] of a cache (bytes): scales equal, codes equal as values."""
    codes, scales = oracle.unpack(cache)
    want_codes, want_scales = oracle.quantise(rows)
    for b in range(len(at)):
        got = codes[b][:, at[b]].transpose(1, 0, 2), scales[b][:, at[b]].transpose(1, 0, 2)
        assert np.array_equal(got[1], want_scales[b])
        ok = ~np.isnan(oracle.values(want_codes[b], want_scales[b]))
        assert np.array_equal(oracle.values(*got)[ok], oracle.values(want_codes[b], want_scales[b])[ok])


def _check_append(c4, B, T, Hq, Hkv, C, position, weights, seed=0):
    qkv, qw, kw = _projection(B, T, Hq, Hkv, seed + 13 * T + C, weights)
    cos, sin = (t.cuda() for t in _tables(C + 3))
    caches = [c4.new_cache(B, Hkv, C).fill_(0xA5) for _ in range(2)]
    dev = [x if x is None else x.cuda() for x in (qkv, qw, kw)]
    q = c4.append(dev[0], cos, sin, position, *caches, dev[1], dev[2], EPS)
    first = np.broadcast_to(np.asarray(position.cpu() if torch.is_tensor(position) else position), (B,))
    at = first[:, None] + np.arange(T)
    ref, mag, k, v = _reference(qkv, qw, kw, at, Hq, Hkv)
    _check_q(q, ref, mag)
    for cache, rows in zip(caches, (k, v)):
        cache = cache.cpu().numpy()
        _check_rows(cache, rows, at)
        # Every other row is as it was.
        codes, scales = oracle.unpack(cache)
        for b in range(B):
            codes[b][:, at[b]], scales[b][:, at[b]] = 5, 0xA5
        assert ((codes == 5) | (codes == 10)).all() and (scales == 0xA5).all()
    assert _status() == 0


@pytest.mark.parametrize("B,T,Hq,Hkv,C,position,weights", [
    (1, 1, 1, 1, 1, 0, None),
    (1, 1, 12, 12, 512, 300, "bf16"),
    (2, 3, 12, 12, 40, 14, "bf16"),       # across a block's end
    (3, 5, 6, 2, 33, 28, "f32"),          # to the last row of an odd capacity
    (2, 16, 4, 1, 64, 16, None),          # exactly one block
    (1, 17, 9, 1, 50, 15, "bf16"),
    (2, 130, 3, 3, 200, 37, "f32"),
    (5, 1, 12, 4, 100, "each", "bf16"),
    (3, 7, 8, 2, 100, "each", None),
    (4, 2, 2, 2, 64, "one", "f32"),
    (1, 515, 32, 8, 600, 5, "bf16"),      # several heads to a warp
])
def test_append_matches_oracle(c4, B, T, Hq, Hkv, C, position, weights):
    if position == "each":
        position = torch.tensor([(31 * b) % (C - T + 1) for b in range(B)], device="cuda")
    elif position == "one":
        position = torch.tensor([C - T - 1], device="cuda")
    _check_append(c4, B, T, Hq, Hkv, C, position, weights)


@pytest.mark.parametrize("kind", ["weights", "table", "large", "small", "no eps"])
def test_append_where_fp32_cannot_decide(c4, kind):
    """Rows for which the FP32 bound says little or FP32 leaves its range: codes as from 64 bits all the same."""
    B, T, H, C = 2, 40, 3, 64
    qkv, qw, kw = _projection(B, T, H, H, 77, "f32")
    cos, sin = _tables(C)
    eps = EPS
    if kind == "weights":        # coefficients of a pair far apart, features the other way round: sums that cancel
        big = torch.arange(64) % 2 == 0
        kw = torch.where(big, kw * 2.0 ** 12, kw * 2.0 ** -12)
        qkv[:, :, H:2 * H] = torch.where(big, qkv[:, :, H:2 * H] * 2.0 ** -12, qkv[:, :, H:2 * H] * 2.0 ** 12)
    elif kind == "table":        # not a rotation: every first element of a pair nearly cancels
        cos, sin = torch.ones(C, 32), torch.ones(C, 32)
        qkv[..., 1::2] = qkv[..., 0::2]
        kw = torch.ones(64)
        kw[1::2] += 2.0 ** -20
    elif kind == "large":
        qkv = (qkv.float() * 2.0 ** 70).to(torch.bfloat16)
    else:
        qkv = (qkv.float() * 2.0 ** -80).to(torch.bfloat16)
        eps = 0.0 if kind == "no eps" else 1e-30
    caches = [c4.new_cache(B, H, C) for _ in range(2)]
    c4.append(qkv.cuda(), cos.cuda(), sin.cuda(), 5, *caches, qw.cuda(), kw.cuda(), eps)
    at = np.broadcast_to(5 + np.arange(T), (B, T))
    k, _ = oracle.norm_rope(_np(qkv[:, :, H:2 * H]), _np(kw), _np(cos)[at], _np(sin)[at], eps)
    _check_rows(caches[0].cpu().numpy(), torch.from_numpy(k).to(torch.bfloat16).double().numpy(), at)


def test_append_layouts_give_the_same_bytes(c4):
    """A 5-D projection, strided and unaligned views, transposed caches, views of larger caches."""
    B, T, H, C = 2, 9, 3, 48
    qkv, qw, kw = (x.cuda() for x in _projection(B, T, H, H, 5))
    cos, sin = (t.cuda() for t in _tables(C))

    def run(x, caches):
        q = c4.append(x, cos, sin, 11, *caches, qw, kw, EPS)
        return [q, *(c.contiguous() for c in caches)]

    want = run(qkv, [c4.new_cache(B, H, C) for _ in range(2)])
    wide = torch.zeros(B, T + 2, 3 * H + 4, 64, dtype=torch.bfloat16, device="cuda")
    wide[:, 1:T + 1, 2:3 * H + 2] = qkv
    odd = torch.zeros(qkv.numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view_as(qkv).copy_(qkv)
    gap = torch.zeros(B, T, 3 * H, 128, dtype=torch.bfloat16, device="cuda")[..., ::2].copy_(qkv)
    for x in (qkv.view(B, T, 3, H, 64), wide[:, 1:T + 1, 2:3 * H + 2], odd, gap,
              qkv.transpose(0, 1).contiguous().transpose(0, 1)):
        assert all(map(torch.equal, want, run(x, [c4.new_cache(B, H, C) for _ in range(2)])))
    turned = [torch.zeros(B, C // 16, H, 576, dtype=torch.uint8, device="cuda").transpose(1, 2) for _ in range(2)]
    inside = [torch.zeros(B + 1, H + 2, C // 16 + 3, 576, dtype=torch.uint8, device="cuda")[1:, 1:H + 1, :C // 16]
              for _ in range(2)]
    for caches in (turned, inside):
        assert all(map(torch.equal, want, run(qkv, caches)))


def test_append_is_norm_rope_then_the_quantiser(c4, fused):
    B, T, Hq, Hkv = 2, 70, 6, 2
    qkv, qw, kw = (x.cuda() for x in _projection(B, T, Hq, Hkv, 8))
    cos, sin = (t.cuda() for t in _tables(200))
    caches = [c4.new_cache(B, Hkv, 100) for _ in range(2)]
    q = c4.append(qkv, cos, sin, 20, *caches, qw, kw, EPS)
    q2, k2, v2 = fused.qkv_norm_rope(qkv, qw, kw, cos, sin, 20, EPS, Hkv)
    assert torch.equal(q, q2) and v2.data_ptr() == qkv[:, :, Hq + Hkv:].data_ptr()
    got = c4.read(*caches, 20, T)
    # k2 is rounded from FP32: the same bf16 number but for a few in 2^-11; v is the same.
    assert torch.equal(got[1].double().cpu(), torch.from_numpy(oracle.values(*oracle.quantise(_np(v2)))))
    same = got[0].double().cpu() == torch.from_numpy(oracle.values(*oracle.quantise(_np(k2))))
    assert same.double().mean() > 0.99


def test_quantiser_on_every_bf16_number(c4):
    """Every finite bf16 number, next to sixteen different largest ones: ties, subnormals, saturation, zeros."""
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    every = every[every.isfinite()]
    rows = []
    for i in range(16):
        x = every[torch.randperm(len(every), generator=torch.Generator().manual_seed(i))]
        rows.append(x[:len(x) // 64 * 64].view(-1, 64))
        # Numbers near each other, so that codes are not all zero: sorted by magnitude.
        y = x[:len(x) // 16 * 16].float().abs().sort().values.to(torch.bfloat16).view(-1, 16)
        sign = torch.randint(0, 2, y.shape, generator=torch.Generator().manual_seed(i)) * 2 - 1
        y = (y * sign)[torch.randperm(len(y), generator=torch.Generator().manual_seed(i))]
        rows.append(y[:len(y) // 4 * 4].reshape(-1, 64))
    # A tie of every scale: the largest 6 s, others border x s.
    top = torch.arange(8, 16).float()[:, None] * torch.exp2(torch.arange(-17, 10).float())
    ties = torch.tensor([6, .25, -.25, .75, 1.25, -1.25, 1.75, 2.5, 3.5, -3.5, 5, -5, .5, 0, -6, 4])
    rows.append((top.reshape(-1, 1) * ties).to(torch.bfloat16).reshape(-1, 64))
    v = torch.cat(rows)
    T = len(v)
    qkv = torch.zeros(1, T, 3, 64, dtype=torch.bfloat16)
    qkv[0, :, 2] = v
    cos, sin = (torch.zeros(T, 32, device="cuda") for _ in range(2))
    caches = [c4.new_cache(1, 1, T) for _ in range(2)]
    c4.append(qkv.cuda(), cos, sin, 0, *caches)
    _check_rows(caches[1].cpu().numpy(), _np(v)[None, :, None], np.arange(T)[None])
    back = c4.read(*caches, 0, T)[1]
    codes, scales = oracle.unpack(caches[1].cpu().numpy())
    assert np.array_equal(_np(back)[0, 0], oracle.values(codes, scales)[0, 0, :T])


def test_quantiser_of_values_that_are_not_finite(c4):
    inf, nan = float("inf"), float("nan")
    v = torch.ones(4, 64)
    v[0, 3] = nan
    v[1, 20], v[1, 21] = inf, -inf
    v[2, 40], v[2, 41] = inf, nan
    v[3] = 0
    qkv = torch.zeros(1, 4, 3, 64)
    qkv[0, :, 2] = v
    cos, sin = (t.cuda() for t in _tables(4))
    caches = [c4.new_cache(1, 1, 4) for _ in range(2)]
    c4.append(qkv.to(torch.bfloat16).cuda(), cos, sin, 0, *caches)
    back = c4.read(*caches, 0, 4)[1][0, 0].float().cpu()
    # Ones: 1/6 = 1.333 * 2^-3 is rounded to 1.375 * 2^-3, and the code is a six: 1.03125.
    assert back[0, :16].isnan().all() and (back[0, 16:] == 1.03125).all()
    assert back[1, 20] == 61440 and back[1, 21] == -61440 and (back[1, 22:32] == 0).all()
    assert back[2, 32:48].isnan().all() and (back[3] == 0).all()


def test_append_outside_the_cache_or_table_is_skipped(c4):
    B, T, H = 4, 3, 2
    qkv, qw, kw = (x.cuda() for x in _projection(B, T, H, H, 3))
    cos, sin = (t.cuda() for t in _tables(40))
    caches = [c4.new_cache(B, H, 32).fill_(7) for _ in range(2)]
    _status()
    for far in (2**63 - 1, -2**63, 2**31, 2**32 + 3):
        before = [c.clone() for c in caches]
        q = c4.append(qkv, cos, sin, torch.tensor([far], device="cuda"), *caches, qw, kw, EPS)
        assert _status() == 2 and (q == 0).all() and all(map(torch.equal, before, caches))
    at = torch.tensor([-2, 30, 2**62, 5], device="cuda")
    q = c4.append(qkv, cos, sin, at, *caches, qw, kw, EPS)
    assert _status() == 2
    ok = [[2], [0, 1], [], [0, 1, 2]]
    for b in range(B):
        for t in range(T):
            assert (q[b, :, t] != 0).any().item() == (t in ok[b])
        rows = [at[b].item() + t for t in ok[b]]
        codes, _ = oracle.unpack(caches[1][b:b + 1].cpu().numpy())
        touched = [r for r in range(32) if not ((codes[0, :, r] == 7) | (codes[0, :, r] == 0)).all()]
        assert touched == rows
    # A table shorter than the cache.
    caches = [c4.new_cache(1, H, 64) for _ in range(2)]
    c4.append(qkv[:1], cos, sin, torch.tensor([39], device="cuda"), *caches, qw, kw, EPS)
    assert _status() == 2 and c4.read(*caches, 39, 1)[1].abs().sum() > 0 and c4.read(*caches, 40, 2)[1].abs().sum() == 0


def _random_cache(B, H, C, seed, spread=0.5):
    """Bytes and values of a random cache of ceil(C / 16) blocks."""
    rs = np.random.RandomState(seed)
    n = -(-C // 16) * 16
    codes = rs.randint(0, 16, (B, H, n, 64))
    scales = np.clip(np.round(8 * (15 + np.log2(0.3) + spread * rs.randn(B, H, n, 4))), 0, 0xE2).astype(np.uint8)
    return oracle.pack(codes, scales), oracle.values(codes, scales)


@pytest.mark.parametrize("B,H,C,start,rows", [(1, 1, 1, 0, 1), (2, 3, 40, 13, 20), (3, 2, 100, 0, 100),
                                              (1, 5, 1000, 333, 600), (2, 1, 64, "each", 7), (2, 2, 64, "one", 16)])
def test_read_is_exact(c4, B, H, C, start, rows):
    kb, kv = _random_cache(B, H, C, C)
    vb, vv = _random_cache(B, H, C, C + 1, spread=4)
    vb.reshape(-1)[:512] = np.arange(512) % 256     # every byte
    vv = oracle.values(*oracle.unpack(vb))
    first = np.zeros(B, int)
    if start == "each":
        first = np.array([5 * b + 1 for b in range(B)])
        start = torch.from_numpy(first).cuda()
    elif start == "one":
        first[:] = 40
        start = torch.tensor([40], device="cuda")
    else:
        first[:] = start
    k, v = torch.from_numpy(kb).cuda(), torch.from_numpy(vb).cuda()
    got = c4.read(k, v, start, rows)
    turned = c4.read(k.transpose(1, 2).contiguous().transpose(1, 2), v.clone(), start, rows)
    for g, t, want in zip(got, turned, (kv, vv)):
        want = np.stack([want[b][:, first[b]:first[b] + rows] for b in range(B)])
        assert np.array_equal(_np(g), want, equal_nan=True) and torch.equal(g, t)


def test_read_outside_the_cache_is_zero(c4):
    kb, vb = (_random_cache(2, 1, 32, s)[0] for s in (1, 2))
    k, v = torch.from_numpy(kb).cuda(), torch.from_numpy(vb).cuda()
    _status()
    got = c4.read(k, v, torch.tensor([-1, 30], device="cuda"), 3)
    assert _status() == 2
    all_k = c4.read(k, v, 0, 32)[0]
    assert (got[0][0, 0, 0] == 0).all() and torch.equal(got[0][0, 0, 1:], all_k[0, 0, :2])
    assert (got[0][1, 0, 2] == 0).all() and torch.equal(got[0][1, 0, :2], all_k[1, 0, 30:])
    for far in (2**63 - 1, 2**63 - 2, -2**63, 2**31, 2**32 + 5, -2**32 + 1):
        got = c4.read(k, v, torch.tensor([far, 0], device="cuda"), 20)
        assert _status() == 2
        assert (got[0][0] == 0).all() and (got[1][0] == 0).all() and torch.equal(got[0][1], all_k[1, :, :20])
    for start in range(-20, 33):          # every way to lie across the ends, and across blocks
        got = c4.read(k, v, torch.tensor([start], device="cuda"), 21)
        for i in range(21):
            want = all_k[:, :, start + i] if 0 <= start + i < 32 else torch.zeros_like(all_k[:, :, 0])
            assert torch.equal(got[0][:, :, i], want)
    _status()
    for bad in (-1, 30):
        with pytest.raises(RuntimeError, match="capacity"):
            c4.read(k, v, bad, 3)


def _queries(B, Hq, T, seed):
    return torch.randn(B, Hq, T, 64, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)


def _check_attention(c4, q, kb, vb, kv, vv, lens):
    dev = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    args = (q.cuda(), torch.from_numpy(kb).cuda(), torch.from_numpy(vb).cuda(), dev)
    o, lse = c4.attention_with_lse(*args)
    C = kv.shape[2]
    ref, ref_lse, A = oracle.attention(_np(q), kv, vv, [C] * len(q) if lens is None else lens)
    got, got_lse = _np(o), _np(lse)
    empty = np.isneginf(ref_lse)
    assert (got[empty] == 0).all() and np.isneginf(got_lse[empty]).all()
    err = np.abs(got - ref)
    S = np.nan_to_num(np.abs(vv)).sum(2, keepdims=True).repeat(q.shape[1] // vv.shape[1], axis=1)
    assert (err <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -9 * A + 2.0 ** -32 * S).all(), err.max()
    lerr = np.abs(got_lse[~empty] - ref_lse[~empty])
    assert (lerr <= 2.0 ** -12 + 2.0 ** -20 * np.abs(ref_lse[~empty])).all(), lerr.max()
    # Without LSE, and once more: the same bits.
    assert torch.equal(o, c4.attention(*args))


@pytest.mark.parametrize("B,Hq,Hkv,T,C,lens", [
    (1, 1, 1, 1, 1, [1]),
    (3, 2, 2, 1, 64, [0, 1, 64]),
    (4, 3, 3, 1, 100, [15, 16, 17, 63]),         # ends inside blocks and tiles
    (2, 12, 12, 1, 300, None),
    (5, 2, 2, 1, 130, [-3, 0, 64, 65, 1000]),    # lengths are clamped
    (2, 4, 1, 1, 500, [499, 250]),
    (2, 8, 1, 1, 500, [500, 128]),
    (2, 9, 1, 1, 200, [200, 3]),                 # nine rows: the 16-row tile
    (1, 16, 1, 1, 700, [650]),
    (1, 24, 1, 1, 260, [259]),                   # two row tiles, the second half full
    (3, 2, 2, 2, 90, [1, 2, 90]),                # a query that sees nothing
    (3, 2, 1, 4, 90, [3, 67, 90]),
    (2, 6, 2, 5, 200, [129, 64]),
    (2, 3, 1, 7, 150, [150, 70]),                # 21 rows
    (2, 2, 2, 16, 300, [290, 10]),
    (1, 9, 1, 16, 140, [133]),                   # 144 rows, nine tiles
    (1, 1, 1, 1, 9000, [8999]),                  # one sequence over many CTAs
    (1, 4, 2, 3, 20001, [20000]),
    (2, 2, 1, 1, 40000, [39999, 5]),             # several clusters, one sequence nearly empty
    (70, 2, 2, 1, 1100, None),
])
def test_attention_matches_oracle(c4, B, Hq, Hkv, T, C, lens):
    kb, kv = _random_cache(B, Hkv, C, 3 * C + T)
    vb, vv = _random_cache(B, Hkv, C, 5 * C + T)
    _check_attention(c4, _queries(B, Hq, T, C), kb, vb, kv, vv, lens)


@pytest.mark.parametrize("B,Hq,Hkv,T", [(160, 1, 1, 1), (80, 2, 2, 1), (160, 4, 1, 1), (150, 4, 1, 3), (40, 8, 4, 5),
                                        (300, 1, 1, 2)])
def test_attention_many_sequences(c4, B, Hq, Hkv, T):
    """Many sequences with room for long ones: empty, short and a few long ones, their tiles in equal shares for all
    warps. What is behind the lengths is NaN."""
    blocks, rows = 450, 1600
    rs = np.random.RandomState(B + T)
    lens = rs.randint(0, 200, B)
    lens[[0, 1, B - 1]] = 0
    lens[[5, B // 2]] = rows, 1111
    kb, kv = _random_cache(B, Hkv, rows, 71)
    vb, vv = _random_cache(B, Hkv, rows, 72)
    full = [torch.full((B, Hkv, blocks, 576), 0xFF, dtype=torch.uint8, device="cuda") for _ in range(2)]
    for dst, src in zip(full, (kb, vb)):
        codes, scales = oracle.unpack(src)
        for b, n in enumerate(lens):
            scales[b, :, n:] = 0xFF
        dst[:, :, :rows // 16] = torch.from_numpy(oracle.pack(codes, scales)).cuda()
    q = _queries(B, Hq, T, 73)
    for order in (np.arange(B), np.argsort(lens)):
        dev = torch.from_numpy(lens[order]).cuda()
        args = (q[order].cuda(), *(x[order] for x in full), dev)
        o, lse = c4.attention_with_lse(*args)
        ref, ref_lse, A = oracle.attention(_np(q)[order], kv[order], vv[order], lens[order])
        S = np.abs(vv[order]).sum(2, keepdims=True).repeat(Hq // Hkv, axis=1)
        got, got_lse = _np(o), _np(lse)
        empty = np.isneginf(ref_lse)
        assert (got[empty] == 0).all() and np.isneginf(got_lse[empty]).all()
        assert (np.abs(got - ref) <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -9 * A + 2.0 ** -32 * S).all()
        lerr = np.abs(got_lse[~empty] - ref_lse[~empty])
        assert (lerr <= 2.0 ** -12 + 2.0 ** -20 * np.abs(ref_lse[~empty])).all()
        assert torch.equal(o, c4.attention(*args))
    # Nothing to see at all.
    o, lse = c4.attention_with_lse(*args[:3], torch.zeros(B, dtype=torch.int32, device="cuda"))
    assert (o == 0).all() and torch.isneginf(lse).all()


@pytest.mark.parametrize("B,Hq,Hkv,T", [(513, 1, 1, 1), (513, 4, 2, 3), (1700, 2, 1, 1), (5000, 1, 1, 1)])
def test_attention_thousands_of_sequences(c4, B, Hq, Hkv, T):
    """More sequences than a count of 32 or of a CTA's threads, runs of empty ones longer than both, and sequences of
    several tiles on either side of each multiple of 32."""
    rows, blocks = 160, 4 * (24576 // (B * Hkv) + 2)
    rs = np.random.RandomState(B + T)
    kb, kv = _random_cache(B, Hkv, rows, 81)
    vb, vv = _random_cache(B, Hkv, rows, 82)
    full = [torch.full((B, Hkv, blocks, 576), 0xFF, dtype=torch.uint8, device="cuda") for _ in range(2)]
    for dst, src in zip(full, (kb, vb)):
        dst[:, :, :rows // 16] = torch.from_numpy(src).cuda()
    q = _queries(B, Hq, T, 83)
    S = np.abs(vv).sum(2, keepdims=True).repeat(Hq // Hkv, axis=1)
    for kind in range(4):
        lens = rs.randint(0, 20, B)
        lens[::32] = 160
        lens[31::64] = 65
        if kind == 1:
            lens[:500] = 0                    # a share begins far behind the first sequence
        if kind == 2:
            lens[7:-3] = 0                    # nearly nothing between the two ends
        if kind == 3:
            lens[5:] = 0
        args = (q.cuda(), *full, torch.from_numpy(lens).cuda())
        o, lse = c4.attention_with_lse(*args)
        ref, ref_lse, A = oracle.attention(_np(q), kv, vv, lens)
        got, got_lse = _np(o), _np(lse)
        empty = np.isneginf(ref_lse)
        assert (got[empty] == 0).all() and np.isneginf(got_lse[empty]).all()
        assert (np.abs(got - ref) <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -9 * A + 2.0 ** -32 * S).all()
        lerr = np.abs(got_lse[~empty] - ref_lse[~empty])
        assert (lerr <= 2.0 ** -12 + 2.0 ** -20 * np.abs(ref_lse[~empty])).all()
        assert torch.equal(o, c4.attention(*args))


def test_attention_weights_reach_every_row(c4):
    """One row at a time has all the weight: a wrong row, feature or scale shows."""
    C, H = 400, 1
    kb, kv = _random_cache(1, H, C, 1)
    vb, vv = _random_cache(1, H, C, 2, spread=2)
    at = [0, 1, 7, 8, 15, 16, 31, 63, 64, 100, 255, 256, 333, 398, 399]
    codes, scales = oracle.unpack(kb)
    q = torch.zeros(len(at), 1, 1, 64)
    kbs = np.repeat(kb, len(at), 0)
    for i, row in enumerate(at):
        c, s = codes.copy(), scales.copy()
        s[...] = 0x40                                 # 2^-7
        s[0, 0, row] = 0x88                           # 4
        q[i, 0, 0] = torch.from_numpy(np.sign(oracle.values(c, s)[0, 0, row])) * 8
        kbs[i] = oracle.pack(c, s)[0]
    kvs = oracle.values(*oracle.unpack(kbs))
    _check_attention(c4, q.to(torch.bfloat16), kbs, np.repeat(vb, len(at), 0), kvs, np.repeat(vv, len(at), 0),
                     [C] * len(at))


@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** -20, 1.0, 2.0 ** 10])
def test_attention_query_magnitudes(c4, scale):
    """Queries over bf16's range (large ones against small keys, so that scores stay below the tolerance's bound)."""
    B, H, C = 2, 2, 200
    kb, _ = _random_cache(B, H, C, 9)
    codes, scales = oracle.unpack(kb)
    if scale > 1:
        scales = np.maximum(scales.astype(int) - 80, 0).astype(np.uint8)   # keys 2^-10
    kb = oracle.pack(codes, scales)
    vb, vv = _random_cache(B, H, C, 10)
    q = (_queries(B, H, 1, 11).float() * scale).to(torch.bfloat16)
    q[0, 0, 0, 1:] *= 2.0 ** -12                     # one element above the others
    _check_attention(c4, q, kb, vb, oracle.values(codes, scales), vv, [200, 77])


def test_attention_rising_scores(c4):
    """Scores that rise along the cache in small steps and in leaps: the running maximum moves, or lags behind."""
    C = 1000
    for slope in (0.02, 0.5, -0.5):
        kb, kv = _random_cache(1, 1, C, 21)
        codes, scales = oracle.unpack(kb)
        codes[..., 0] = 2                              # 1.0, times a scale that goes with the row
        rows = 32 * (0.5 + 0.5 * np.arange(C + 8) / C) if slope > 0 else 32 * (1 - 0.5 * np.arange(C + 8) / C)
        codes[..., 1:16] = 0
        scales[0, 0, :, 0] = oracle.nearest(rows, oracle.SCALES)
        kb, kv = oracle.pack(codes, scales), oracle.values(codes, scales)
        vb, vv = _random_cache(1, 1, C, 22)
        q = torch.zeros(1, 1, 1, 64)
        q[..., 0] = 8 * abs(slope)
        _check_attention(c4, q.to(torch.bfloat16), kb, vb, kv, vv, [C])


def test_attention_ignores_what_is_not_seen(c4):
    """NaN scales and codes behind the lengths, and in rows that only some of the queries see."""
    B, Hq, Hkv, T, C = 3, 4, 2, 5, 200
    kb, kv = _random_cache(B, Hkv, C, 31)
    vb, vv = _random_cache(B, Hkv, C, 32)
    lens = [130, 64, 3]
    q = _queries(B, Hq, T, 33)
    dev = torch.tensor(lens, device="cuda")
    want = c4.attention_with_lse(q.cuda(), torch.from_numpy(kb).cuda(), torch.from_numpy(vb).cuda(), dev)
    for cache in (kb, vb):
        codes, scales = oracle.unpack(cache)
        for b, n in enumerate(lens):
            scales[b, :, n:] = 0xFF
            codes[b, :, n:] = 15
        cache[...] = oracle.pack(codes, scales)
    got = c4.attention_with_lse(q.cuda(), torch.from_numpy(kb).cuda(), torch.from_numpy(vb).cuda(), dev)
    assert all(map(torch.equal, want, got))
    # The last row of each sequence is NaN in one group of V and in K: the last query alone sees it.
    codes, scales = oracle.unpack(vb)
    for b, n in enumerate(lens):
        scales[b, :, n - 1, 2] = 0xFF
    vb2 = oracle.pack(codes, scales)
    o = c4.attention(q.cuda(), torch.from_numpy(kb).cuda(), torch.from_numpy(vb2).cuda(), dev)
    assert torch.equal(o[:, :, :-1], want[0][:, :, :-1])
    assert o[:, :, -1, 32:48].isnan().all()
    assert torch.equal(o[:, :, -1, :32], want[0][:, :, -1, :32])
    assert torch.equal(o[:, :, -1, 48:], want[0][:, :, -1, 48:])
    codes, scales = oracle.unpack(kb)
    for b, n in enumerate(lens):
        scales[b, :, n - 1, 1] = 0xFF
    o = c4.attention(q.cuda(), torch.from_numpy(oracle.pack(codes, scales)).cuda(), torch.from_numpy(vb).cuda(), dev)
    assert torch.equal(o[:, :, :-1], want[0][:, :, :-1]) and o[:, :, -1].isnan().all()


def test_attention_queries_that_are_not_finite(c4):
    kb, _ = _random_cache(1, 2, 100, 41)
    vb, _ = _random_cache(1, 2, 100, 42)
    k, v = torch.from_numpy(kb).cuda(), torch.from_numpy(vb).cuda()
    q = _queries(1, 4, 2, 43).cuda()
    want = c4.attention(q, k, v)
    q[0, 1, 0, 5], q[0, 2, 1, 9] = float("nan"), float("inf")
    got = c4.attention(q, k, v)
    assert got[0, 1, 0].isnan().all() and got[0, 2, 1].isnan().all()
    keep = torch.ones(4, 2, dtype=torch.bool)
    keep[1, 0] = keep[2, 1] = False
    assert torch.equal(got[0][keep], want[0][keep])


def test_attention_layouts(c4):
    B, Hq, Hkv, T, C = 2, 6, 2, 3, 150
    k, v = (torch.from_numpy(_random_cache(B, Hkv, C, s)[0]).cuda() for s in (51, 52))
    q = _queries(B, Hq, T, 53).cuda()
    lens = torch.tensor([150, 40], device="cuda")
    want = c4.attention(q, k, v, lens)
    strided = q.transpose(1, 2).contiguous().transpose(1, 2)
    odd = torch.zeros(q.numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view_as(q).copy_(q)
    wide = torch.zeros(B, Hq, T, 128, dtype=torch.bfloat16, device="cuda")[..., ::2].copy_(q)
    turned = k.transpose(1, 2).contiguous().transpose(1, 2)
    big = torch.zeros(B, Hkv + 1, k.shape[2] + 2, 576, dtype=torch.uint8, device="cuda")
    big[:, 1:, 1:-1] = v
    for x in (strided, odd, wide):
        assert torch.equal(want, c4.attention(x, turned, big[:, 1:, 1:-1], lens))
    # A shorter view of the same storage.
    short = c4.attention(q, k[:, :, :4], v[:, :, :4], torch.tensor([64, 40], device="cuda"))
    assert torch.equal(short[1], want[1])


@pytest.mark.parametrize("bad,match", [
    (lambda q, k, v: (q.float(), k, v), "bf16"),
    (lambda q, k, v: (q[..., :32], k, v), "head_dim=64"),
    (lambda q, k, v: (q[:, :3], k, v), "multiple"),
    (lambda q, k, v: (q[:1], k, v), "batch size"),
    (lambda q, k, v: (q, k, v[:, :, :1]), "same shape"),
    (lambda q, k, v: (q, k[..., :560], v[..., :560]), "576"),
    (lambda q, k, v: (q, k.float(), v), "uint8"),
    (lambda q, k, v: (q.expand(-1, -1, 17, -1), k, v), "16 query tokens"),
    (lambda q, k, v: (q, k, v, torch.zeros(3, dtype=torch.int32, device="cuda")), "shape"),
    (lambda q, k, v: (q, k, v, torch.zeros(2, device="cuda")), "int32 or int64"),
    (lambda q, k, v: (q, k, v, torch.zeros(2, dtype=torch.int32)), "same device"),
    (lambda q, k, v: (q, k.cpu(), v), "CUDA"),
    (lambda q, k, v: (q, k.view(-1)[:0].view(2, 2, 0, 576), v.view(-1)[:0].view(2, 2, 0, 576)), "positive"),
])
def test_attention_refusals(c4, bad, match):
    q, k = _queries(2, 4, 1, 1).cuda(), c4.new_cache(2, 2, 32)
    with pytest.raises(RuntimeError, match=match):
        c4.attention(*bad(q, k, k.clone()))


@pytest.mark.parametrize("change,match", [
    (dict(qkv=lambda x: x.float()), "bf16"),
    (dict(qkv=lambda x: x[..., :32]), "head_dim=64"),
    (dict(qkv=lambda x: x[:, :, :4]), "multiple"),
    (dict(qkv=lambda x: x[:, :, :7]), "multiple"),
    (dict(qkv=lambda x: x[:1]), "batch size"),
    (dict(qkv=lambda x: x[:, :0]), "positive"),
    (dict(cos=lambda x: x[:, :16]), "tables"),
    (dict(cos=lambda x: x[:10]), "same shape"),
    (dict(sin=lambda x: x.double()), "tables"),
    (dict(position=lambda x: 30), "capacity"),
    (dict(position=lambda x: -1), "table"),
    (dict(position=lambda x: torch.zeros(3, dtype=torch.long, device="cuda")), "one element"),
    (dict(position=lambda x: torch.zeros(2, 3, dtype=torch.long, device="cuda")), "one element"),
    (dict(position=lambda x: torch.zeros(1, dtype=torch.int32, device="cuda")), "int64"),
    (dict(position=lambda x: torch.zeros(1, dtype=torch.long)), "int64 CUDA"),
    (dict(cos=lambda x: x.cpu()), "CUDA"),
    (dict(position=lambda x: 1.5), "int or an int64"),
    (dict(cache_k=lambda x: x[:, :1]), "multiple|same shape"),
    (dict(cache_k=lambda x: x.to(torch.int8)), "uint8"),
    (dict(cache_k=lambda x: x, cache_v="cache_k"), "caches of their own"),
    (dict(q_weight=lambda x: None), "both norm weights"),
    (dict(q_weight=lambda x: x.float()), "both be"),
    (dict(k_weight=lambda x: x[:32]), "shape"),
    (dict(eps=lambda x: -1.0), "eps"),
])
def test_append_refusals(c4, change, match):
    qkv, qw, kw = (x.cuda() for x in _projection(2, 3, 4, 2, 1))
    cos, sin = (t.cuda() for t in _tables(64))
    args = dict(qkv=qkv, cos=cos, sin=sin, position=0, cache_k=c4.new_cache(2, 2, 32),
                cache_v=c4.new_cache(2, 2, 32), q_weight=qw, k_weight=kw, eps=EPS)
    for key, f in change.items():
        args[key] = args[f] if isinstance(f, str) else f(args[key])
    with pytest.raises(RuntimeError, match=match):
        c4.append(**args)


def test_inference_only(c4):
    qkv, qw, kw = (x.cuda() for x in _projection(2, 3, 4, 2, 1))
    cos, sin = (t.cuda() for t in _tables(64))
    q, k, v = _queries(2, 4, 1, 1).cuda(), c4.new_cache(2, 2, 32), c4.new_cache(2, 2, 32)
    calls = [(lambda: c4.append(qkv, cos, sin, 0, k, v, qw, kw, EPS), (qkv, cos, qw, kw)),
             (lambda: c4.attention(q, k, v), (q,)), (lambda: c4.attention_with_lse(q, k, v), (q,)),
             (lambda: c4.read(k, v, 0, 1), ())]
    for call, tensors in calls:
        with torch.autocast("cuda", torch.bfloat16), pytest.raises(RuntimeError, match="AMP"):
            call()
        for t in tensors:
            t.requires_grad_()
            with pytest.raises(NotImplementedError, match="no backward"):
                call()
            with torch.no_grad():
                call()
            t.requires_grad_(False)


def test_offsets_past_32_bits(c4):
    """A cache of more than 2^32 bytes: the last sequence is written, read and attended to."""
    B, H, blocks = 3, 2, 1300000
    k = torch.empty(B, H, blocks, 576, dtype=torch.uint8, device="cuda")     # 4.5 GB
    v = torch.empty_like(k)
    rows, T = 300, 4
    C = blocks * 16
    small = [c4.new_cache(1, H, 320) for _ in range(2)]
    qkv, qw, kw = (x.cuda() for x in _projection(B, rows, H, H, 3))
    cos, sin = (t.cuda() for t in _tables(rows))
    cos, sin = (torch.cat([torch.ones(1, 32, device="cuda").expand(16, 32), t]) for t in (cos, sin))
    # The rows lie at the front of the last sequence's heads, and (a view) at the very end of the cache.
    for big in (k, v):
        big[2, :, :20] = 0
    c4.append(qkv[2:], cos, sin, 3, *small, qw, kw, EPS)
    c4.append(qkv, cos, sin, 3, k[:, :, :20], v[:, :, :20], qw, kw, EPS)
    assert all(torch.equal(a[0], b[2, :, :20]) for a, b in zip(small, (k, v)))
    for a, b in zip(small, (k, v)):
        b[2, :, blocks - 20:] = a[0]
    got = c4.read(k[2:], v[2:], C - 320, 320)
    assert all(map(torch.equal, got, c4.read(*small, 0, 320)))
    q = _queries(1, H, T, 4).cuda()
    want = c4.attention(q, *small)
    assert torch.equal(c4.attention(q, k[2:, :, blocks - 20:], v[2:, :, blocks - 20:]), want)
    # The whole of the last sequence: 20.8 million rows, of which only the last have a key that is not zero.
    k[2, :, :blocks - 20] = 0
    v[2, :, :blocks - 20] = 0
    o, lse = c4.attention_with_lse(q, k[2:], v[2:])
    ko, vo = (x[0].double() for x in c4.read(*small, 0, 320))
    for t in range(T):
        n = 320 - (T - 1 - t)
        s = torch.einsum("hcd,hd->hc", ko[:, :n], q[0, :, t].double()) / 8
        total = torch.log(s.exp().sum(-1) + (C - 320))
        assert ((lse[0, :, t].double() - total).abs() <= 2.0 ** -12 + 2.0 ** -20 * total).all()
        weight = (s - total[:, None]).exp()
        ref = torch.einsum("hc,hcd->hd", weight, vo[:, :n])
        A = torch.einsum("hc,hcd->hd", weight, vo[:, :n].abs())
        assert ((o[0, :, t].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -9 * A).all()


def test_streams_and_captured_steps(c4):
    """Append and attention in one captured step whose position and lengths move on the device, replayed, on another
    stream, with two graphs sharing the caches: the same bits as eager calls."""
    B, Hq, Hkv, C, steps = 3, 8, 2, 9000, 6
    qkv, qw, kw = (x.cuda() for x in _projection(B, steps, Hq, Hkv, 61))
    cos, sin = (t.cuda() for t in _tables(C))
    start = [torch.from_numpy(_random_cache(B, Hkv, C, s)[0]).cuda() for s in (62, 63)]
    first = torch.tensor([100, 4000, 8990], device="cuda")

    eager = [x.clone() for x in start]
    want = []
    for i in range(steps):
        q = c4.append(qkv[:, i:i + 1], cos, sin, first + i, *eager, qw, kw, EPS)
        want.append(c4.attention(q, *eager, first + i + 1))
    torch.cuda.synchronize()

    caches = [x.clone() for x in start]
    token = torch.empty_like(qkv[:, :1])
    position = first.clone()
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")

    def step():
        lens.copy_(position + 1)
        q = c4.append(token, cos, sin, position, *caches, qw, kw, EPS)
        o = c4.attention(q, *caches, lens)
        position.add_(1)
        return o

    token.copy_(qkv[:, :1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(side):
        step()
        torch.cuda.synchronize()
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                outs.append(step())
            graphs.append(g)
        position.copy_(first)
        for a, b in zip(caches, start):
            a.copy_(b)
        for i in range(steps):
            token.copy_(qkv[:, i:i + 1])
            graphs[i % 2].replay()
            assert torch.equal(outs[i % 2], want[i])
    torch.cuda.synchronize()
    assert all(map(torch.equal, caches, eager))
    assert _status() == 0


def _uneven_cache(q, lens, H, C, seed, share, size, kind):
    """Keys with one row a head that takes about `share` of a single query's weight (0: none), and values of about `size`:
    kind "heavy": the heavy row's value is zero; "small": 2^-6 of the others'; "mixed": rows and groups of sizes from
    2^-8 to 1 of it; "large": a row of no weight has values near 10^4."""
    rs = np.random.RandomState(seed)
    B = len(lens)
    kb, kv = _random_cache(B, H, C, seed)
    codes, scales = oracle.unpack(kb)
    vcodes = rs.randint(0, 16, codes.shape)
    log = np.log2(size / 3) + 0.5 * rs.randn(*scales.shape)
    if kind == "mixed":
        log -= 8 * rs.rand(*scales.shape)
    vscales = np.round(8 * (15 + log))
    for b, n in enumerate(lens):
        for h in range(H):
            x = q[b, h, 0]
            others = np.exp(kv[b, h, :n] @ x / 8).sum()
            heavy, light = rs.choice(n, 2, replace=False)
            codes[b, h, heavy] = np.where(x < 0, 10, 2)      # its key points where the query does
            if share > 0:
                s = np.log(share / (1 - share) * others) / (np.abs(x).sum() / 8)
                scales[b, h, heavy] = oracle.nearest(s, oracle.SCALES)
                if kind == "heavy":
                    vscales[b, h, heavy] = 0
                elif kind == "small":
                    vscales[b, h, heavy] -= 48
            if kind == "large":
                codes[b, h, light] = np.where(x < 0, 2, 10)  # away from it
                scales[b, h, light] = oracle.nearest(12 / (np.abs(x).sum() / 8), oracle.SCALES)
                vscales[b, h, light] = 0xDA
    vscales = np.clip(vscales, 0, 0xE2).astype(np.uint8)
    return (oracle.pack(codes, scales), oracle.pack(vcodes, vscales), oracle.values(codes, scales),
            oracle.values(vcodes, vscales))


SMALL_VALUES = [(0.9, 1.0, "heavy"), (0.9, 0.1, "small"), (0.9, 0.01, "heavy"), (0.9, 1e-3, "small"), (0.5, 1e-2, "heavy"),
                (0.5, 1e-3, "small"), (0.5, 1e-4, "heavy"), (0.999, 0.03, "heavy"), (0, 1e-3, "mixed"), (0, 1e-4, ""),
                (0.9, 0.1, "mixed"), (0, 1e-3, "large"), (0.5, 1.0, "large")]


@pytest.mark.parametrize("B,H,C,flat,share,size,kind", [
    (B, H, C, False, *case) for B, H, C in ((1, 3, 512), (2, 2, 4096), (1, 1, 9000)) for case in SMALL_VALUES
] + [(B, H, C, True, *case) for B, H, C in ((20, 12, 2048), (1800, 1, 100)) for case in SMALL_VALUES[2::3]])
def test_attention_small_values_beside_a_heavy_row(c4, B, H, C, flat, share, size, kind):
    """One query row over values of any size, where one row has most of the weight, in the cluster kernel and the flat
    one; the same token as the second of two queries."""
    lens = [C - 7 * (b % 9) for b in range(B)]
    q = _queries(B, H, 1, C + B)
    kb, vb, kv, vv = _uneven_cache(_np(q), lens, H, C, 7 * C + B, share, size, kind)
    if flat:   # capacity enough for the flat kernel's share of all tiles
        blocks = 4 * (24576 // (B * H) + 2)
        wide = [np.full((B, H, blocks, 576), 0xFF, np.uint8) for _ in range(2)]
        for dst, src in zip(wide, (kb, vb)):
            dst[:, :, :src.shape[2]] = src
        kb, vb = wide
    k, v = torch.from_numpy(kb).cuda(), torch.from_numpy(vb).cuda()
    dev = torch.tensor(lens, dtype=torch.int32, device="cuda")
    o, lse = c4.attention_with_lse(q.cuda(), k, v, dev)
    ref, ref_lse, A = oracle.attention(_np(q), kv, vv, lens)
    S = np.abs(vv).sum(2, keepdims=True)
    bound = 2.0 ** -8 * np.abs(ref) + 2.0 ** -9 * A + 2.0 ** -32 * S
    assert (np.abs(_np(o) - ref) <= bound).all(), (np.abs(_np(o) - ref) / bound).max()
    assert (np.abs(_np(lse) - ref_lse) <= 2.0 ** -12 + 2.0 ** -20 * np.abs(ref_lse)).all()
    two = c4.attention(torch.cat((_queries(B, H, 1, 3), q), 2).cuda(), k, v, dev)
    assert (np.abs(_np(two[:, :, 1:]) - _np(o)) <= 2 * bound).all()


@pytest.mark.parametrize("B,H,C,flat", [(3, 2, 300, False), (1, 1, 9000, False), (160, 1, 200, True)])
def test_attention_of_one_query_sees_keys_that_are_not_numbers(c4, B, H, C, flat):
    """A key group of NaN in a row that a single query sees makes its O and LSE NaN, whatever the query's signs; behind the
    length it changes nothing."""
    kb, _ = _random_cache(B, H, C, 91)
    vb, _ = _random_cache(B, H, C, 92)
    if flat:
        more = ((0, 0), (0, 0), (0, 4 * (24576 // (B * H) + 2) - kb.shape[2]), (0, 0))
        kb, vb = np.pad(kb, more), np.pad(vb, more)
    lens = [C - 1 - b % 5 for b in range(B)]
    v, dev = torch.from_numpy(vb).cuda(), torch.tensor(lens, device="cuda")
    q = _queries(B, H, 1, 93).cuda()
    want = c4.attention_with_lse(q, torch.from_numpy(kb).cuda(), v, dev)
    codes, scales = oracle.unpack(kb)
    for b, n in enumerate(lens):
        scales[b, :, n:] = 0xFF
    behind = c4.attention_with_lse(q, torch.from_numpy(oracle.pack(codes, scales)).cuda(), v, dev)
    assert all(map(torch.equal, want, behind))
    for group, row in ((0, 0), (1, 77), (2, C // 2), (3, lens[0] - 1)):
        bad = scales.copy()
        bad[0, 0, row, group] = 0xFF
        for sign in (1, -1):
            signed = c4.attention_with_lse(sign * q, torch.from_numpy(kb).cuda(), v, dev)
            for x, y in zip(c4.attention_with_lse(sign * q, torch.from_numpy(oracle.pack(codes, bad)).cuda(), v, dev),
                            signed):
                assert x[0, 0].isnan().all()
                keep = torch.ones(B, H, dtype=torch.bool)
                keep[0, 0] = False
                assert torch.equal(x[keep], y[keep])


def test_append_then_attention_of_a_key_that_is_not_a_number(c4):
    """A NaN that append meets in a projection reaches the output of one query and of two."""
    B, T, H = 1, 5, 2
    qkv, qw, kw = (x.cuda() for x in _projection(B, T, H, H, 5))
    qkv[0, 2, H, 9] = float("nan")                # the first head's key of token 2
    cos, sin = (t.cuda() for t in _tables(32))
    caches = [c4.new_cache(B, H, 32) for _ in range(2)]
    q = c4.append(qkv, cos, sin, 0, *caches, qw, kw, EPS)
    lens = torch.tensor([T], device="cuda")
    for tokens in (1, 2):
        o = c4.attention(q[:, :, -tokens:], *caches, lens)
        assert o[0, 0].isnan().all() and o[0, 1].isfinite().all()


def test_append_to_caches_beside_one_another(c4):
    """Keys and values in the gaps of one another's layout; views that overlap are refused and write nothing."""
    B, T, H, n = 2, 9, 3, 3
    qkv, qw, kw = (x.cuda() for x in _projection(B, T, H, H, 5))
    cos, sin = (t.cuda() for t in _tables(16 * n))

    def run(*caches):
        return c4.append(qkv, cos, sin, 11, *caches, qw, kw, EPS)

    want = [c4.new_cache(B, H, 16 * n) for _ in range(2)]
    q = run(*want)
    for shape, dim in (((2, B, H, n, 576), 0), ((B, 2, H, n, 576), 1), ((B, H, 2, n, 576), 2), ((B, H, n, 2, 576), 3),
                       ((B, H, n, 576 * 2), None)):
        both = torch.zeros(shape, dtype=torch.uint8, device="cuda")
        got = both.unbind(dim) if dim is not None else (both[..., 576:], both[..., :576])
        assert torch.equal(run(*got), q) and all(map(torch.equal, got, want))
    row = torch.zeros(4 * B * H * n * 576, dtype=torch.uint8, device="cuda")
    over = row.as_strided((B, H, n, 576), (576, 576, 576, 1))
    heads = row.as_strided((B, H, n, 576), (H * n * 576, (n - 1) * 576, 576, 1))
    plain = row[:B * H * n * 576].view(B, H, n, 576)
    behind = row[576:][:B * H * n * 576].view(B, H, n, 576)
    other = c4.new_cache(B, H, 16 * n)
    for caches, match in (((over, other), "overlap"), ((other, heads), "overlap"),
                          ((plain, behind), "caches of their own"), ((behind, plain), "caches of their own")):
        with pytest.raises(RuntimeError, match=match):
            run(*caches)
    assert (row == 0).all() and (other == 0).all()


def test_forward_mode_derivatives_are_refused(c4):
    import torch.autograd.forward_ad as forward_ad
    qkv, qw, kw = (x.cuda() for x in _projection(2, 3, 4, 2, 1))
    cos, sin = (t.cuda() for t in _tables(64))
    q, k, v = _queries(2, 4, 1, 1).cuda(), c4.new_cache(2, 2, 32), c4.new_cache(2, 2, 32)
    with forward_ad.dual_level():
        for i in range(5):
            x = [qkv, cos, sin, qw, kw]
            x[i] = forward_ad.make_dual(x[i], torch.ones_like(x[i]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                c4.append(*x[:3], 0, k, v, *x[3:], EPS)
        assert (k == 0).all() and (v == 0).all()
        dual = forward_ad.make_dual(q, q)
        for call in (c4.attention, c4.attention_with_lse):
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call(dual, k, v)
