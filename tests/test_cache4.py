"""Query/key norm and 4-bit KV cache without a GPU: argument checks of the C ABI before any CUDA call, guards of
the Python entry points, and the oracle's own definitions."""
import ctypes
import os
import re
from unittest.mock import Mock, patch

import numpy as np
import pytest
import torch

from oracle import cache4_oracle as oracle

BAD_ARG, UNSUPPORTED = 1, 2
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    from tiny_transformer_b200.operators._extension import load_c_abi
    return load_c_abi()


def _s(*s):
    return (ctypes.c_int64 * len(s))(*s)


def _err(lib):
    return lib.tt_attn_last_error().decode()


def _projection(qkv=16, strides=None, B=2, T=5, Hq=4, Hkv=2, qw=16, kw=16, f32=0, cos=16, sin=16, L=100, pos=0,
                dev=None, sb=0):
    heads = Hq + 2 * Hkv
    strides = strides if strides is not None else _s(T * heads * 64, heads * 64, 64)
    return [qkv, strides, B, T, Hq, Hkv, qw, kw, f32, cos, sin, L, pos, dev, sb]


COMMON = [
    (dict(qkv=None), BAD_ARG, "NULL"),
    (dict(cos=None), BAD_ARG, "NULL"),
    (dict(B=0), BAD_ARG, "positive"),
    (dict(Hkv=0), BAD_ARG, "positive"),
    (dict(L=0), BAD_ARG, "positive"),
    (dict(qw=None), BAD_ARG, "both weights"),
    (dict(T=2**31, L=2**40), BAD_ARG, "grid limits"),
    (dict(B=2**28 - 1, T=64, L=100), BAD_ARG, "grid limits"),
    (dict(pos=96), BAD_ARG, "exceeds the cos/sin table"),
    (dict(pos=-1), BAD_ARG, "exceeds the cos/sin table"),
    (dict(pos=2**63 - 1), BAD_ARG, "exceeds the cos/sin table"),
    (dict(sb=-1), BAD_ARG, "negative"),
    (dict(dev=20), BAD_ARG, "8-byte"),
    (dict(kw=24), BAD_ARG, "16-byte"),
    (dict(qw=20, f32=1), BAD_ARG, "16-byte"),
    (dict(sin=8), BAD_ARG, "16-byte"),
    (dict(qkv=24), UNSUPPORTED, "aligned"),
    (dict(strides=_s(5 * 8 * 64 + 4, 8 * 64, 64)), UNSUPPORTED, "multiples of 8"),
    (dict(strides=_s(5 * 8 * 64, 8 * 64, 0)), UNSUPPORTED, "multiples of 8"),
]


@pytest.mark.parametrize("kwargs,status,fragment", COMMON + [
    (dict(q=None), BAD_ARG, "outputs"),
    (dict(k=8), BAD_ARG, "outputs"),
    (dict(eps=-1.0), BAD_ARG, "eps"),
    (dict(eps=float("nan")), BAD_ARG, "eps"),
])
def test_norm_rope_rejects_before_cuda(lib, kwargs, status, fragment):
    kwargs = dict(kwargs)
    q, k, eps = kwargs.pop("q", 16), kwargs.pop("k", 16), kwargs.pop("eps", 1e-6)
    assert lib.tt_attn_qkv_norm_rope_bf16(*_projection(**kwargs), 0, eps, q, k, None) == status
    assert fragment in _err(lib)


@pytest.mark.parametrize("kwargs,status,fragment", COMMON + [
    (dict(dx=None), BAD_ARG, "dqkv"),
    (dict(dqw=None), BAD_ARG, "weights' gradients"),
    (dict(ws=None), BAD_ARG, "workspace"),
    (dict(ws_bytes=8), BAD_ARG, "workspace"),
    (dict(dkw=17), BAD_ARG, "aligned to their type"),
    (dict(g=24), UNSUPPORTED, "gradients need"),
    (dict(gs=None), BAD_ARG, "needs its strides"),
    (dict(gs=_s(4 * 5 * 64, 5 * 64, 128, 2)), UNSUPPORTED, "gradients need"),
])
def test_norm_rope_backward_rejects_before_cuda(lib, kwargs, status, fragment):
    kwargs = dict(kwargs)
    a = {n: kwargs.pop(n, 16) for n in ("g", "dx", "dqw", "dkw", "ws")}
    gs = kwargs.pop("gs", _s(4 * 5 * 64, 5 * 64, 64, 1))
    ws_bytes = kwargs.pop("ws_bytes", 1 << 30)
    assert lib.tt_attn_qkv_norm_rope_backward_bf16(
        *_projection(**kwargs), 0, 1e-6, a["g"], gs, None, None, None, None, a["dx"], a["dqw"], a["dkw"],
        a["ws"], ws_bytes, None) == status
    assert fragment in _err(lib)


def _cache(n=7, H=2):
    return _s(H * n * 576, n * 576, 576, 1)


@pytest.mark.parametrize("kwargs,status,fragment", COMMON + [
    (dict(q=None), BAD_ARG, "NULL"),
    (dict(ck=None), BAD_ARG, "NULL"),
    (dict(n=0), BAD_ARG, "positive"),
    (dict(n=2**30), BAD_ARG, "fit int32"),
    (dict(pos=100, L=1000, n=6), BAD_ARG, "cache capacity"),
    (dict(ck=24), UNSUPPORTED, "caches need"),
    (dict(ck=32), BAD_ARG, "caches of their own"),
    (dict(cs=_s(2 * 7 * 576, 7 * 576, 584, 1)), UNSUPPORTED, "caches need"),
    (dict(cs=_s(2 * 7 * 576, 7 * 576, 576, 2)), UNSUPPORTED, "caches need"),
    (dict(cs=_s(2 * 7 * 576, 7 * 576, 560, 1)), UNSUPPORTED, "at least 576"),   # blocks over one another
    (dict(cs=_s(2 * 7 * 576, 0, 576, 1)), UNSUPPORTED, "at least 576"),
])
def test_append_rejects_before_cuda(lib, kwargs, status, fragment):
    kwargs = dict(kwargs)
    q, ck, n = kwargs.pop("q", 16), kwargs.pop("ck", 16), kwargs.pop("n", 7)
    cs = kwargs.pop("cs", _cache())
    assert lib.tt_attn_cache4_append_bf16(*_projection(**kwargs), 1e-6, q, ck, cs, 32, _cache(), n,
                                          None) == status
    assert fragment in _err(lib)


@pytest.mark.parametrize("kwargs,status,fragment", [
    (dict(ck=None), BAD_ARG, "NULL"),
    (dict(k=8), BAD_ARG, "NULL"),
    (dict(B=0), BAD_ARG, "positive"),
    (dict(rows=0), BAD_ARG, "positive"),
    (dict(start=-1), BAD_ARG, "cache capacity"),
    (dict(start=100, rows=13), BAD_ARG, "cache capacity"),
    (dict(start=2**62), BAD_ARG, "cache capacity"),
    (dict(rows=2**62), BAD_ARG, "grid limits"),
    (dict(B=2**28 - 1), BAD_ARG, "grid limits"),
    (dict(dev=20), BAD_ARG, "8-byte"),
    (dict(sb=-1), BAD_ARG, "negative"),
    (dict(ck=24), UNSUPPORTED, "caches need"),
])
def test_read_rejects_before_cuda(lib, kwargs, status, fragment):
    a = dict(ck=16, B=2, start=0, dev=None, sb=0, rows=5, k=16)
    a.update(kwargs)
    assert lib.tt_attn_cache4_read_bf16(a["ck"], _cache(), 16, _cache(), a["B"], 2, 7, a["start"], a["dev"], a["sb"],
                                        a["rows"], a["k"], 16, None) == status
    assert fragment in _err(lib)


def _attn(lib, *, q=16, ck=16, B=2, Hq=4, Hkv=2, T=3, n=7, d=64, lens=None, out=16, lse=None, qs=None, cs=None,
          ws=None, ws_bytes=1 << 40):
    qs = qs or _s(Hq * T * 64, T * 64, 64, 1)
    cs = cs or _s(Hkv * n * 576, n * 576, 576, 1)
    return lib.tt_attn_cache4_forward_bf16(q, qs, ck, cs, 16, cs, B, Hq, Hkv, T, n, d, lens, out, lse, ws,
                                           ws_bytes, None)


@pytest.mark.parametrize("kwargs,status,fragment", [
    (dict(q=None), BAD_ARG, "NULL"),
    (dict(out=None), BAD_ARG, "NULL"),
    (dict(d=128), BAD_ARG, "head_dim=64"),
    (dict(B=0), BAD_ARG, "positive"),
    (dict(T=0), BAD_ARG, "positive"),
    (dict(n=0), BAD_ARG, "positive"),
    (dict(Hq=3), BAD_ARG, "multiple"),
    (dict(T=17), BAD_ARG, "16 query tokens"),
    (dict(n=2**30), BAD_ARG, "fit int32"),
    (dict(B=2**30), BAD_ARG, "grid limits"),
    (dict(out=24), BAD_ARG, "16-byte"),
    (dict(lens=18), BAD_ARG, "4-byte"),
    (dict(lse=18), BAD_ARG, "4-byte"),
    (dict(q=24), UNSUPPORTED, "aligned"),
    (dict(ck=24), UNSUPPORTED, "caches need"),
    (dict(qs=_s(4 * 3 * 66, 3 * 66, 66, 1)), UNSUPPORTED, "multiples of"),
    (dict(cs=_s(2 * 7 * 576, 7 * 576, 580, 1)), UNSUPPORTED, "caches need"),
    (dict(B=1, Hq=1, Hkv=1, T=1, n=10000), BAD_ARG, "workspace"),
])
def test_attention_rejects_before_cuda(lib, kwargs, status, fragment):
    assert _attn(lib, **kwargs) == status
    assert fragment in _err(lib)


def test_workspace_sizes(lib):
    assert lib.tt_attn_cache4_workspace_size(8, 12, 12, 1, 32) == 0        # a cluster for each sequence
    n = lib.tt_attn_cache4_workspace_size(1, 16, 2, 1, 8192)               # few sequences, a long cache
    assert n > 0 and n % (2 * 8 * 66 * 4) == 0
    n = lib.tt_attn_cache4_workspace_size(64, 12, 12, 1, 512)              # many sequences
    assert n == 64 * 12 * 8 + (64 * 12 + 148 * 16) * 8 * 66 * 4            # a table of the units, records
    for bad in ((0, 1, 1, 1, 1), (1, 3, 2, 1, 1), (1, 1, 1, 17, 1), (1, 1, 1, 1, 0), (2**40, 1, 1, 1, 1)):
        assert lib.tt_attn_cache4_workspace_size(*bad) == 0
    assert lib.tt_attn_qkv_norm_rope_backward_workspace_size() % (64 * 4) == 0


def test_format_constants_agree():
    from tiny_transformer_b200.operators import cache4
    header = open(os.path.join(ROOT, "include", "tt_attention.h")).read()
    source = open(os.path.join(ROOT, "tiny-transformer_b200", "csrc", "cache4_sm100.cuh")).read()
    name = {"BLOCK_ROWS": cache4.BLOCK_ROWS, "BLOCK_BYTES": cache4.BLOCK_BYTES,
            "MAX_QUERIES": cache4.MAX_QUERIES}
    for key, value in name.items():
        assert int(re.search(rf"TT_ATTN_CACHE4_{key} (\d+)", header).group(1)) == value
    for key in ("BLOCK_ROWS", "MAX_QUERIES"):
        assert int(re.search(rf"constexpr int {key} = (\d+);", source).group(1)) == name[key]
    byte = int(re.search(r"MAX_SCALE_BYTE = (0x\w+);", source).group(1), 16)
    assert oracle.SCALES[byte] == 10240 and len(oracle.SCALES) == byte + 1


def test_entry_points_forward_to_the_native_module():
    from tiny_transformer_b200.operators import cache4, fused
    t = [object() for _ in range(7)]
    ext = Mock()
    with patch.object(cache4, "load_attention_extension", return_value=ext):
        assert cache4.attention(*t[:3], 5) is ext.cache4_attention.return_value
        ext.cache4_attention.assert_called_with(*t[:3], 5)
        assert cache4.attention_with_lse(*t[:3]) is ext.cache4_attention_with_lse.return_value
        ext.cache4_attention_with_lse.assert_called_with(*t[:3], None)
        cache4.append(t[0], t[1], t[2], 9, t[3], t[4], t[5], t[6], eps=1e-5)
        ext.cache4_append.assert_called_with(t[0], t[1], t[2], 9, t[3], t[4], t[5], t[6], 1e-5)
        cache4.read(t[3], t[4], 2, 3)
        ext.cache4_read.assert_called_with(t[3], t[4], 2, 3)
    with patch.object(fused, "load_attention_extension", return_value=ext):
        fused.qkv_norm_rope(*t[:5], kv_heads=4)
        ext.qkv_norm_rope.assert_called_with(*t[:5], 0, 1e-6, 4)


def test_cpu_tensors_are_refused():
    from tiny_transformer_b200.operators import cache4, fused
    cache = cache4.new_cache(2, 3, 33, device="cpu")
    assert cache.shape == (2, 3, 3, 576)
    x, table, q = torch.zeros(2, 1, 3, 3, 64), torch.zeros(4, 32), torch.zeros(2, 3, 1, 64)
    for call in (lambda: cache4.attention(q, cache, cache), lambda: cache4.attention_with_lse(q, cache, cache),
                 lambda: cache4.read(cache, cache, 0, 1),
                 lambda: cache4.append(x, table, table, 0, cache, cache),
                 lambda: fused.qkv_norm_rope(x, None, None, table, table)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    for bad in ((0, 1, 1), (1, 0, 1), (1, 1, 0)):
        with pytest.raises(ValueError, match="positive"):
            cache4.new_cache(*bad, device="cpu")


def test_oracle_quantiser_is_nearest_and_round_trips():
    rs = np.random.RandomState(3)
    x = rs.randn(7, 64) * np.exp(rs.randn(7, 64))
    codes, scales = oracle.quantise(x)
    got = oracle.values(codes, scales)
    scale = np.repeat(oracle.SCALES[scales], 16, axis=-1)
    table = np.concatenate((oracle.MAGNITUDES, -oracle.MAGNITUDES))
    best = np.abs(x[..., None] - table * scale[..., None]).min(-1)
    assert np.allclose(np.abs(got - x), best)
    # What is in the format comes back as it is, when its group holds a six.
    again = oracle.values(*oracle.quantise(np.where(np.arange(64) % 16 == 0, 6 * scale, got)))
    assert np.array_equal(again, np.where(np.arange(64) % 16 == 0, 6 * scale, got))
    cache = oracle.pack(np.tile(codes[:1, None, None], (2, 3, 32, 1)), np.tile(scales[:1, None, None], (2, 3, 32, 1)))
    back = oracle.unpack(cache)
    assert cache.shape == (2, 3, 2, 576) and np.array_equal(back[0][1, 2, 31], codes[0])
    assert np.array_equal(back[1][0, 1, 5], scales[0])


def test_oracle_gradient_against_differences():
    rs = np.random.RandomState(4)
    x, w, g = rs.randn(1, 2, 2, 64), 1 + 0.2 * rs.randn(64), rs.randn(1, 2, 2, 64)
    angle = rs.rand(1, 2, 32) * 6
    cos, sin = np.cos(angle), np.sin(angle)

    def loss(x, w):
        return (oracle.norm_rope(x, w, cos, sin, 1e-6)[0] * g).sum()

    dx, dw, _, _ = oracle.norm_rope_backward(x, w, cos, sin, 1e-6, g)
    h = 1e-6
    for at in ((0, 0, 0, 0), (0, 1, 1, 63), (0, 1, 0, 30)):
        d = np.zeros_like(x)
        d[at] = h
        assert abs((loss(x + d, w) - loss(x - d, w)) / (2 * h) - dx[at]) < 1e-7
    for i in (0, 31, 63):
        d = np.zeros_like(w)
        d[i] = h
        assert abs((loss(x, w + d) - loss(x, w - d)) / (2 * h) - dw[i]) < 1e-7


ROW = 576


@pytest.mark.parametrize("ks,vs,apart,status,fragment", [
    ((ROW, ROW, ROW), None, 1 << 20, UNSUPPORTED, "overlap"),                      # all blocks of all heads in one row
    ((14 * ROW, 6 * ROW, ROW), None, 1 << 20, UNSUPPORTED, "overlap"),             # a head's last block, the next one's first
    ((14 * ROW - 16, 7 * ROW, ROW), None, 1 << 20, UNSUPPORTED, "overlap"),
    ((7 * ROW, 8 * ROW, ROW), None, 1 << 20, UNSUPPORTED, "overlap"),              # heads outside, sequences too close
    ((2**62, 2**61, 2**60), None, 1 << 20, UNSUPPORTED, "overlap"),                # no such memory
    (None, (ROW, ROW, ROW), 1 << 20, UNSUPPORTED, "overlap"),
    (None, None, ROW, BAD_ARG, "caches of their own"),                             # values one block behind the keys
    (None, None, 7 * ROW, BAD_ARG, "caches of their own"),
    (None, None, 28 * ROW - 16, BAD_ARG, "caches of their own"),
    (None, None, 16, BAD_ARG, "caches of their own"),
    ((28 * ROW, 14 * ROW, 2 * ROW), None, 28 * ROW, BAD_ARG, "caches of their own"),
    ((28 * ROW, 14 * ROW, 2 * ROW), (28 * ROW, 14 * ROW, 2 * ROW), 16, BAD_ARG, "caches of their own"),
])
@pytest.mark.parametrize("first", ["keys", "values"])
def test_append_refuses_caches_over_one_another(lib, ks, vs, apart, status, fragment, first):
    """Blocks that share bytes would be written by different warps in no order."""
    strides = [_s(*(x or (14 * ROW, 7 * ROW, ROW)), 1) for x in (ks, vs)]
    base = [1 << 30, (1 << 30) + apart]
    if first == "values":
        strides.reverse()
        base.reverse()
    assert lib.tt_attn_cache4_append_bf16(*_projection(), 1e-6, 16, base[0], strides[0], base[1], strides[1], 7,
                                          None) == status
    assert fragment in _err(lib)
