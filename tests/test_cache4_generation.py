"""The decoder with a query/key norm and with a 4-bit KV cache: training, eager and graphed generation."""
from dataclasses import replace

import numpy as np
import pytest
import torch

from oracle import cache4_oracle as oracle
from tiny_transformer_b200.generation import (Decoder, DecoderConfig, GraphedDecode, KVCache, KVCache4, generate,
                                              request, rms_norm)
from tiny_transformer_b200.speculative_generation import TokenTree, allocate, forward_tree

SMALL = DecoderConfig(vocab_size=512, dim=128, n_layers=2, n_heads=2, hidden_dim=256, max_seq_len=256,
                      qk_norm=True)


def _model(config=SMALL, backend="reference", dtype=torch.float32, device="cpu", seed=3):
    torch.manual_seed(seed)
    model = Decoder(config, backend).to(device=device, dtype=dtype).eval()
    with torch.no_grad():
        for name, p in model.named_parameters():
            if name.endswith(("q_norm", "k_norm")):
                p.add_(0.2 * torch.randn(64, generator=torch.Generator().manual_seed(7)).to(p))
    return model


def _ids(shape, seed, device="cpu"):
    return torch.randint(0, SMALL.vocab_size, shape, generator=torch.Generator().manual_seed(seed)).to(device)


def test_model_without_norm_is_as_it_was():
    """No new parameter and the same weights from the same seed."""
    plain = _model(replace(SMALL, qk_norm=False))
    normed = _model()
    assert not [n for n, _ in plain.named_parameters() if "_norm" in n and n.split(".")[-1] in ("q_norm", "k_norm")]
    extra = dict(normed.named_parameters())
    for name, p in plain.named_parameters():
        assert torch.equal(p, extra[name])


@torch.inference_mode()
def test_norm_reaches_every_path_cpu():
    model = _model()
    ids = _ids((2, 12), 5)
    full = model(ids)
    cache = model.new_cache(2, 12)
    steps = [model(ids[:, :8], cache=cache)] + [model(ids[:, t:t + 1], cache=cache) for t in range(8, 12)]
    assert torch.allclose(torch.cat(steps, dim=1), full, atol=1e-5, rtol=1e-4)
    block = model.blocks[0]
    q = torch.randn(1, 2, 3, 64)
    assert torch.equal(block.norm_heads(q, q)[1], rms_norm(q, block.k_norm, SMALL.norm_eps))
    # The tree pass of speculative generation, a chain, against the full forward.

    class Ops:
        @staticmethod
        def tree_attention(q, tk, tv, ck, cv, parents, lens):
            n = int(lens[0])
            k, v = torch.cat([ck[:, :, :n], tk], 2), torch.cat([cv[:, :, :n], tv], 2)
            mask = torch.ones(q.shape[2], n + q.shape[2], dtype=torch.bool).tril(n)
            s = (q @ k.transpose(-1, -2) / 8).masked_fill(~mask, float("-inf"))
            return torch.softmax(s, -1) @ v

    cache = model.new_cache(2, 12)
    allocate(model, cache)
    model(ids[:, :8], cache=cache)
    tree = TokenTree((1, 1, 1))
    logits, _, _ = forward_tree(model, ids[:, 8:], tree.parents, tree.depths, cache,
                                torch.full((2,), 8, dtype=torch.int32), Ops)
    assert torch.allclose(logits, full[:, 8:], atol=1e-5, rtol=1e-4)


def test_cache_choice_and_refusals_cpu():
    model = _model()
    assert isinstance(model.new_cache(2, 12), KVCache)
    cache = model.new_cache(2, 40, bits=4)
    assert isinstance(cache, KVCache4) and cache.allocated_bytes() == 0
    keys, values = cache.storage_for(1, 2, torch.device("cpu"))
    assert keys.shape == (2, 2, 3, 576) and cache.allocated_bytes() == 2 * keys.numel()
    assert cache.storage_for(1, 2, torch.device("cpu"))[0] is keys
    with pytest.raises(ValueError, match="device"):
        cache.storage_for(1, 2, torch.device("meta"))
    with pytest.raises(ValueError, match="16 or 4"):
        model.new_cache(2, 12, bits=8)
    for bad in ((0, 12), (2, 0), (2, 257)):
        with pytest.raises(ValueError, match="invalid"):
            model.new_cache(*bad, bits=4)
    with pytest.raises(ValueError, match="head_dim"):
        KVCache4(replace(SMALL, n_heads=4), 1, 8)
    with torch.inference_mode(), pytest.raises(ValueError, match="student"):
        model(_ids((2, 3), 1), cache=cache)
    with torch.inference_mode(), pytest.raises(ValueError, match="capacity"):
        model(_ids((2, 41), 1), cache=cache)


def _gpu():
    if not torch.cuda.is_available() or torch.cuda.get_device_capability()[0] != 10:
        pytest.skip("needs an sm_100 GPU")


@pytest.mark.gpu
def test_training_with_norm_gpu():
    """Loss and gradients of the student decoder (norm, rotation and attention kernels) against the reference
    attention in FP32: bf16 rounding in every operator, so within a few per cent of each gradient's norm."""
    _gpu()
    ids = _ids((3, 40), 1, "cuda")

    def grads(backend, dtype):
        model = _model(SMALL, backend, dtype, "cuda").train()
        logits = model(ids).float()
        loss = torch.nn.functional.cross_entropy(logits[:, :-1].flatten(0, 1), ids[:, 1:].flatten())
        loss.backward()
        return loss.item(), {n: p.grad.double() for n, p in model.named_parameters()}

    want, wg = grads("reference", torch.float32)
    got, gg = grads("student", torch.bfloat16)
    same, sg = grads("reference", torch.bfloat16)
    assert abs(got - want) < 2e-2
    for name, g in wg.items():
        # No worse than three times what the reference's own bf16 run is off (and 2 % where that is tiny).
        bound = 3 * (sg[name] - g).norm() + 0.02 * g.norm()
        assert (gg[name] - g).norm() <= bound, name
    assert all(gg[f"blocks.{i}.{n}"].abs().sum() > 0 for i in range(2) for n in ("q_norm", "k_norm"))


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("qk_norm", [True, False])
def test_norm_decode_matches_reference_gpu(qk_norm):
    """The 16-bit cache: eager and graphed decode of a model with the norm."""
    _gpu()
    model = _model(replace(SMALL, qk_norm=qk_norm), "student", torch.bfloat16, "cuda")
    ids = _ids((3, 40), 1, "cuda")
    model.set_attention("reference")
    want = model(ids).float()
    model.set_attention("student")
    assert (model(ids).float() - want).abs().max().item() < 3e-2
    cache = model.new_cache(3, 40)
    inc = [model(ids[:, :24], cache=cache)] + [model(ids[:, t:t + 1], cache=cache) for t in range(24, 40)]
    assert (torch.cat(inc, 1).float() - want).abs().max().item() < 3e-2
    assert torch.equal(generate(model, ids, 12), generate(model, ids, 12, graphed=True))


class _QuantisedUpdate(KVCache):
    """A 16-bit cache whose rows are rounded to what a 4-bit one would hold."""

    def update(self, layer, k, v):
        rows = [torch.from_numpy(oracle.values(*oracle.quantise(x.double().cpu().numpy()))).to(x) for x in (k, v)]
        return super().update(layer, *rows)


@pytest.mark.gpu
@torch.inference_mode()
def test_cache4_logits_gpu():
    """A decoder over a 4-bit cache gives the logits of one whose 16-bit cache is rounded to the same values, whatever
    the prompt is cut into."""
    _gpu()
    model = _model(SMALL, "student", torch.bfloat16, "cuda")
    ids = _ids((3, 60), 2, "cuda")
    cache = _QuantisedUpdate(SMALL, 3, 60)
    want = [model(ids[:, :37], cache=cache)] + [model(ids[:, t:t + 1], cache=cache) for t in range(37, 60)]
    want = torch.cat(want, 1).float()
    for cuts in ([60], [37] + [1] * 23, [1] * 60, [20, 5, 16, 17, 2]):
        cache = model.new_cache(3, 60, bits=4)
        out, at = [], 0
        for n in cuts:
            out.append(model(ids[:, at:at + n], cache=cache))
            at += n
        assert cache.length == 60
        assert (torch.cat(out, 1).float() - want).abs().max().item() < 3e-2, cuts
    assert cache.allocated_bytes() == 2 * 2 * 3 * 2 * 4 * 576


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("qk_norm", [True, False])
def test_cache4_generation_gpu(qk_norm):
    """Eager and captured steps generate the same tokens; request() runs on it."""
    _gpu()
    model = _model(replace(SMALL, qk_norm=qk_norm), "student", torch.bfloat16, "cuda")
    prompt = _ids((4, 20), 3, "cuda")
    eager = generate(model, prompt, 30, cache_bits=4)
    graphed = generate(model, prompt, 30, graphed=True, cache_bits=4)
    assert eager.shape == (4, 30) and torch.equal(eager, graphed)
    r = request(model, prompt, 12, graphed=True, cache_bits=4)
    assert torch.equal(r["last_tokens"], eager[:, :12]) and r["kv_allocated_bytes"] == 2 * 2 * 4 * 2 * 2 * 576
    cache = model.new_cache(4, 24, bits=4)
    first = model(prompt, cache=cache, last_only=True)[:, -1].argmax(-1, keepdim=True)
    g = GraphedDecode(model, cache, 4)
    g.prepare(first)
    g.capture()
    g.replay(3)
    with pytest.raises(ValueError, match="output buffer|capacity"):
        g.replay(8)
    torch.cuda.synchronize()
    assert np.array_equal(g.tokens().cpu().numpy(), eager[:, :4].cpu().numpy())
