"""Speculative-decoding operators without a GPU: argument checks of the C ABI before any CUDA call,
guards of the Python entry points, and the oracle's own definition."""
import ctypes
from unittest.mock import Mock, patch

import numpy as np
import pytest
import torch

from oracle import speculative_oracle as oracle

BAD_ARG, UNSUPPORTED = 1, 2


@pytest.fixture(scope="module")
def lib():
    from tiny_transformer_b200.operators._extension import load_c_abi
    return load_c_abi()


def _s(*s):
    return (ctypes.c_int64 * 4)(*s)


def _err(lib):
    return lib.tt_attn_last_error().decode()


def _tree(lib, *, q=16, tk=16, tv=16, ck=16, cv=16, B=2, Hq=4, Hkv=2, N=5, C=100, d=64, parents=16,
          ps=0, lens=None, out=16, lse=None, qs=None, cs=None, ws=None, ws_bytes=1 << 40):
    qs = qs or _s(Hq * N * 64, N * 64, 64, 1)
    ts = _s(Hkv * N * 64, N * 64, 64, 1)
    cs = cs or _s(Hkv * C * 64, C * 64, 64, 1)
    return lib.tt_attn_tree_forward_bf16(q, qs, tk, ts, tv, ts, ck, cs, cv, cs, B, Hq, Hkv, N, C, d,
                                         parents, ps, lens, out, lse, ws, ws_bytes, None)


@pytest.mark.parametrize("kwargs,status,fragment", [
    (dict(q=None), BAD_ARG, "NULL"),
    (dict(parents=None), BAD_ARG, "NULL"),
    (dict(out=None), BAD_ARG, "NULL"),
    (dict(d=128), BAD_ARG, "head_dim=64"),
    (dict(B=0), BAD_ARG, "positive"),
    (dict(N=0), BAD_ARG, "positive"),
    (dict(C=0), BAD_ARG, "positive"),
    (dict(Hq=3), BAD_ARG, "multiple"),
    (dict(N=257), BAD_ARG, "256 nodes"),
    (dict(C=2**31), BAD_ARG, "fit int32"),
    (dict(ps=4), BAD_ARG, "parents_stride"),
    (dict(ps=-1), BAD_ARG, "parents_stride"),
    (dict(B=2**30), BAD_ARG, "grid limits"),
    (dict(out=24), BAD_ARG, "16-byte"),
    (dict(parents=18), BAD_ARG, "4-byte"),
    (dict(lens=17), BAD_ARG, "4-byte"),
    (dict(lse=18), BAD_ARG, "4-byte"),
    (dict(q=24), UNSUPPORTED, "aligned"),
    (dict(cs=_s(2 * 100 * 66, 100 * 66, 66, 1)), UNSUPPORTED, "multiples of 8"),
    (dict(cs=_s(2 * 100 * 128, 100 * 128, 128, 2)), UNSUPPORTED, "unit last stride"),
])
def test_tree_forward_rejects_before_cuda(lib, kwargs, status, fragment):
    assert _tree(lib, **kwargs) == status
    assert fragment in _err(lib)


def _verify(lib, *, tokens=16, parents=16, ps=0, p=16, psb=50, psn=10, q=None, qsb=0, qsn=0, u=16, B=2,
            N=5, V=10, path=16, counts=16, nxt=16):
    return lib.tt_attn_tree_verify_f32(tokens, parents, ps, p, psb, psn, q, qsb, qsn, u, B, N, V, path,
                                       counts, nxt, None)


@pytest.mark.parametrize("kwargs,fragment", [
    (dict(tokens=None), "NULL"),
    (dict(nxt=None), "NULL"),
    (dict(B=0), "positive"),
    (dict(V=0), "positive"),
    (dict(N=257), "256 nodes"),
    (dict(V=(1 << 22) + 1), "4194304"),
    (dict(B=2**30), "grid limits"),
    (dict(ps=3), "parents_stride"),
    (dict(psb=-1), "negative"),
    (dict(p=18), "4-byte"),
    (dict(tokens=20), "8-byte"),
])
def test_verify_rejects_before_cuda(lib, kwargs, fragment):
    assert _verify(lib, **kwargs) == BAD_ARG
    assert fragment in _err(lib)


def _commit(lib, *, ck=16, tk=16, layers=2, B=2, H=2, N=4, C=10, d=64, path=16, P=3, counts=16, lens=16,
            new=32, cs=None, null_list=False):
    ptrs = lambda x: (ctypes.c_void_p * max(layers, 1))(*[x] * max(layers, 1))  # noqa: E731
    cs = cs or _s(H * C * 64, C * 64, 64, 1)
    ts = _s(H * N * 64, N * 64, 64, 1)
    return lib.tt_attn_tree_commit_bf16(None if null_list else ptrs(ck), cs, ptrs(16), cs, ptrs(tk), ts,
                                        ptrs(16), ts, layers, B, H, N, C, d, path, P, counts, lens,
                                        new, None)


@pytest.mark.parametrize("kwargs,status,fragment", [
    (dict(null_list=True), BAD_ARG, "NULL"),
    (dict(ck=None), BAD_ARG, "NULL"),
    (dict(path=None), BAD_ARG, "NULL"),
    (dict(layers=0), BAD_ARG, "positive"),
    (dict(P=0), BAD_ARG, "positive"),
    (dict(d=32), BAD_ARG, "head_dim=64"),
    (dict(B=2**30), BAD_ARG, "grid limits"),
    (dict(new=16), BAD_ARG, "buffer of its own"),
    (dict(counts=18), BAD_ARG, "4-byte"),
    (dict(tk=24), UNSUPPORTED, "aligned"),
    (dict(cs=_s(2 * 10 * 68, 10 * 68, 68, 1)), UNSUPPORTED, "multiples of 8"),
])
def test_commit_rejects_before_cuda(lib, kwargs, status, fragment):
    assert _commit(lib, **kwargs) == status
    assert fragment in _err(lib)


def test_header_limits_match_the_kernels():
    import os
    import re
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    header = open(os.path.join(root, "include", "tt_attention.h")).read()
    src = os.path.join(root, "tiny-transformer_b200", "csrc")
    nodes = int(re.search(r"TT_ATTN_TREE_MAX_NODES (\d+)", header).group(1))
    for name in ("tree_attention_sm100.cuh", "tree_verify_sm100.cuh"):
        text = open(os.path.join(src, name)).read()
        assert int(re.search(r"MAX_NODES = (\d+);", text).group(1)) == nodes
    text = open(os.path.join(src, "tree_verify_sm100.cuh")).read()
    n = {k: int(re.search(rf"constexpr int {k} = (\d+);", text).group(1))
         for k in ("MAX_CLUSTER", "MAX_WINDOWS", "WINDOW")}
    vocab = int(re.search(r"TT_ATTN_TREE_MAX_VOCAB (\d+)", header).group(1))
    assert n["MAX_CLUSTER"] * n["MAX_WINDOWS"] * n["WINDOW"] == vocab


def test_entry_points_forward_and_guard():
    from tiny_transformer_b200.operators import speculative
    ten = [Mock(is_cuda=True, requires_grad=False) for _ in range(5)]
    par, lens, o, lse = object(), object(), object(), object()
    ext = Mock()
    ext.tree_attention.return_value = (o, lse)
    with patch.object(speculative, "load_attention_extension", return_value=ext):
        assert speculative.tree_attention(*ten, par, lens) is o
        ext.tree_attention.assert_called_with(*ten, par, lens, False)
        assert speculative.tree_attention_with_lse(*ten, par) == (o, lse)
        ext.tree_attention.assert_called_with(*ten, par, None, True)
        speculative.commit_path(ten[0], [ten[1]], (ten[2],), ten[3], 1, 2, 3)
        ext.tree_commit.assert_called_with([ten[0]], [ten[1]], [ten[2]], [ten[3]], 1, 2, 3)
        with patch.object(torch, "is_autocast_enabled", return_value=True), \
                pytest.raises(RuntimeError, match="AMP"):
            speculative.tree_attention(*ten, par)
        for x in ten:
            x.requires_grad = True
            with pytest.raises(NotImplementedError, match="backward"):
                speculative.tree_attention(*ten, par)
            with torch.no_grad():
                assert speculative.tree_attention(*ten, par) is o
            x.requires_grad = False
            x.is_cuda = False
            with pytest.raises(RuntimeError, match="CUDA"):
                speculative.tree_attention(*ten, par)
            x.is_cuda = True


def test_native_rejects_cpu_tensors():
    from tiny_transformer_b200.operators import speculative
    from tiny_transformer_b200.operators._extension import load_attention_extension
    x = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16)
    par = torch.tensor([-1, 0])
    with pytest.raises(RuntimeError, match="CUDA"):
        load_attention_extension().tree_attention(x, x, x, x, x, par)
    with pytest.raises(RuntimeError, match="CUDA"):
        speculative.verify_tree(par[None], par, torch.ones(1, 2, 3), torch.ones(1, 2))
    with pytest.raises(RuntimeError, match="CUDA"):
        speculative.commit_path(x, x, x, x, par[None], par[:1], par[:1])


def test_oracle_chains():
    assert oracle.chains([-1, 0, 0, 2, -2, 4, 6, 1 << 30, -1]) == [
        [0], [1, 0], [2, 0], [3, 2, 0], [], [], [], [], [8]]


def test_oracle_tree_attention_of_a_chain_is_causal_attention():
    from oracle import attention_oracle
    rs = np.random.RandomState(0)
    q, k, v = (rs.randn(1, 2, 12, 64) for _ in range(3))
    chain = np.arange(-1, 4)[None]
    o, lse, _ = oracle.tree_attention(q[:, :, 7:], k[:, :, 7:], v[:, :, 7:], k[:, :, :7], v[:, :, :7],
                                      chain, [7])
    want, want_lse = attention_oracle.attention_fp64(q[:, :, 7:], k, v, 7)
    assert np.allclose(o, want, atol=1e-12) and np.allclose(lse, want_lse, atol=1e-12)


def test_oracle_walk_follows_the_target_distribution():
    """First token after the root over 40000 walks with two tries (drawn children): Pearson's
    statistic with 3 degrees of freedom below 35 (probability above it 1.2e-7)."""
    rs, B, V = np.random.RandomState(1), 40000, 4
    p, q = np.array([0.1, 0.5, 0.25, 0.15]), np.array([0.4, 0.2, 0.2, 0.2])
    tokens = np.concatenate([np.zeros((B, 1), int), rs.choice(V, (B, 2), p=q)], 1)
    rows = lambda x: np.broadcast_to(x.astype(np.float32), (B, 3, V))  # noqa: E731
    path, counts, nxt = oracle.verify_tree(tokens, np.tile([[-1, 0, 0]], (B, 1)), rows(p),
                                           rs.rand(B, 3).astype(np.float32), rows(q))
    first = np.where(counts > 1, np.take_along_axis(tokens, np.maximum(path[:, 1:2], 0), 1)[:, 0], nxt)
    seen = np.bincount(first, minlength=V)
    assert ((seen - p * B) ** 2 / (p * B)).sum() < 35


def test_every_cuda_failure_is_reported_by_the_helper_that_clears_it():
    """A failed launch leaves its error pending in the runtime; a return that does not read it makes the
    next call report it as its own."""
    import os
    import re
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "tiny-transformer_b200", "csrc")
    abi = open(os.path.join(csrc, "tt_attention_abi.cu")).read()
    text = abi + open(os.path.join(csrc, "speculative_abi.cuh")).read()
    helper = re.search(r"tt_attn_status cuda_fail\(.*?\n}\n", abi, re.S).group(0)
    assert "cudaGetLastError()" in helper and "cudaGetErrorString" in helper
    assert text.count("cudaGetErrorString") == 1
    # What a launch call returns goes to the check that reads the pending error too.
    launches = re.findall(r"cudaLaunchKernelEx\(", text)
    assert len(launches) > 0 and len(re.findall(r"check_launch\(\"[^\"]+\", le\)", text)) == 6
