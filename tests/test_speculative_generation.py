"""Speculative generation: the host logic on CPU with the operators replaced by their 64-bit
restatements, and the three operators together on the GPU."""
import types

import numpy as np
import pytest
import torch

from oracle import speculative_oracle as oracle
from tiny_transformer_b200.generation import Decoder, DecoderConfig, generate
from tiny_transformer_b200.speculative_generation import (TokenTree, allocate, forward_tree,
                                                          generate_speculative)

SMALL = DecoderConfig(vocab_size=96, dim=128, n_layers=2, n_heads=2, hidden_dim=128, max_seq_len=128)


def _cpu_ops():
    def tree_attention(q, tk, tv, ck, cv, parents, lens):
        p = np.broadcast_to(parents.numpy(), (q.shape[0], q.shape[2]))
        args = [x.double().numpy() for x in (q, tk, tv, ck, cv)]
        return torch.from_numpy(oracle.tree_attention(*args, p, lens.numpy())[0]).to(q.dtype)

    def verify_tree(tokens, parents, p, u, q=None):
        par = np.broadcast_to(parents.numpy(), tokens.shape)
        out = oracle.verify_tree(tokens.numpy(), par, p.numpy(), u.numpy(),
                                 None if q is None else q.numpy())
        return tuple(torch.from_numpy(x) for x in out)

    def commit_path(ck, cv, tk, tv, path, counts, lens):
        for b in range(len(counts)):
            n, at = int(counts[b]), int(lens[b])
            for c, t in zip(ck + cv, tk + tv):
                c[b, :, at:at + n] = t[b][:, path[b, :n].long()]
        return (lens + counts).int()

    return types.SimpleNamespace(tree_attention=tree_attention, verify_tree=verify_tree,
                                 commit_path=commit_path)


def _model(seed, dtype=torch.float32, device="cpu", backend="reference", config=SMALL):
    torch.manual_seed(seed)
    model = Decoder(config, backend).to(device=device, dtype=dtype).eval()
    with torch.no_grad():
        model.embedding.mul_(10)  # peaked distributions
    return model


def _prompt(batch, time, device="cpu", seed=1):
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(0, SMALL.vocab_size, (batch, time), generator=gen).to(device)


def test_token_tree_is_in_level_order():
    tree = TokenTree((2, 1, 3))
    assert tree.parents.tolist() == [-1, 0, 0, 1, 2, 3, 3, 3, 4, 4, 4]
    assert tree.depths.tolist() == [0, 1, 1, 2, 2, 3, 3, 3, 3, 3, 3]
    assert tree.levels == [(0, 1), (1, 3), (3, 5), (5, 11)] and tree.size == 11 and tree.depth == 3
    with pytest.raises(ValueError):
        TokenTree((2, 0))


@torch.inference_mode()
def test_forward_tree_matches_plain_forward_cpu():
    """Logits of every node are those of a plain forward over the prompt and the node's branch."""
    model, prompt = _model(3), _prompt(2, 7)
    tree = TokenTree((2, 2))
    cache = model.new_cache(2, 16)
    allocate(model, cache)
    model(prompt[:, :-1], cache=cache, last_only=True)
    ids = torch.cat([prompt[:, -1:], _prompt(2, tree.size - 1, seed=5)], 1)
    lens = torch.full((2,), 6, dtype=torch.int32)
    logits, _, _ = forward_tree(model, ids, tree.parents, tree.depths, cache, lens, _cpu_ops())
    for n in range(tree.size):
        chain = oracle.chains(tree.parents.tolist())[n][::-1]
        full = torch.cat([prompt[:, :-1], ids[:, chain]], 1)
        assert torch.allclose(logits[:, n], model(full)[:, -1], atol=2e-4, rtol=1e-3)


@pytest.mark.parametrize("time,branching", [(1, (1,)), (6, (3, 2)), (9, (1, 1, 1, 1))])
def test_greedy_speculation_gives_the_greedy_tokens_cpu(time, branching):
    model, draft, prompt = _model(3), _model(4), _prompt(3, time)
    want = generate(model, prompt, 11)
    got, stats = generate_speculative(model, draft, prompt, 11, branching, temperature=0,
                                      ops=_cpu_ops())
    assert torch.equal(got, want)
    assert 1 <= stats["accepted"] <= len(branching) + 1


def test_a_draft_that_is_the_target_is_accepted_whole_cpu():
    model, prompt = _model(3), _prompt(2, 5)
    want = generate(model, prompt, 12)
    got, stats = generate_speculative(model, model, prompt, 12, (1, 1, 1), temperature=0,
                                      ops=_cpu_ops())
    assert torch.equal(got, want) and stats["steps"] == 3


def test_sampling_is_reproducible_cpu():
    model, draft, prompt = _model(3), _model(4), _prompt(2, 4)
    runs = [generate_speculative(model, draft, prompt, 9, (2, 2), 1.0,
                                 torch.Generator().manual_seed(7), _cpu_ops())[0] for _ in range(2)]
    assert torch.equal(*runs) and runs[0].shape == (2, 9)


def test_refusals():
    model, prompt = _model(3), _prompt(1, 4)
    with pytest.raises(ValueError, match="positive"):
        generate_speculative(model, model, prompt, 0, ops=_cpu_ops())
    with pytest.raises(ValueError, match="negative"):
        generate_speculative(model, model, prompt, 3, temperature=-1.0, ops=_cpu_ops())
    with pytest.raises(ValueError, match="max_seq_len"):
        generate_speculative(model, model, prompt, 200, ops=_cpu_ops())
    other = _model(3, config=DecoderConfig(vocab_size=64, dim=128, n_layers=1, n_heads=2,
                                           hidden_dim=128, max_seq_len=128))
    with pytest.raises(ValueError, match="vocabulary"):
        generate_speculative(model, other, prompt, 3, ops=_cpu_ops())


def _gpu():
    if not torch.cuda.is_available() or torch.cuda.get_device_capability()[0] != 10:
        pytest.skip("needs an sm_100 GPU")


@pytest.mark.gpu
@pytest.mark.parametrize("temperature,branching", [(0, (3, 2, 1)), (1.0, (2, 2)), (0, (4, 4, 1))])
@torch.inference_mode()
def test_speculation_on_the_gpu(temperature, branching):
    """The operators together. Greedy: every token is the most probable one of a plain forward, up to
    the bf16 noise of its logits, two units in the last place of the largest."""
    _gpu()
    model = _model(3, torch.bfloat16, "cuda", "student")
    draft = _model(4, torch.bfloat16, "cuda", "student")
    prompt = _prompt(4, 10, "cuda")
    got, stats = generate_speculative(model, draft, prompt, 24, branching, temperature,
                                      torch.Generator("cuda").manual_seed(3))
    assert got.shape == (4, 24) and 1 <= stats["accepted"] <= len(branching) + 1
    assert ((got >= 0) & (got < SMALL.vocab_size)).all()
    if temperature == 0:
        logits = model(torch.cat([prompt, got], 1))[:, prompt.shape[1] - 1:-1].float()
        gap = logits.amax(-1) - logits.gather(-1, got[..., None])[..., 0]
        unit = 2.0 ** (torch.floor(torch.log2(logits.abs().max())).item() - 7)
        assert gap.max().item() <= 2 * unit
    # A draft that is the target is accepted whole, but for the noise between two passes.
    _, stats = generate_speculative(model, model, prompt, 24, (1, 1, 1), temperature,
                                    torch.Generator("cuda").manual_seed(3))
    assert stats["accepted"] > 2.5


@pytest.mark.parametrize("time,new_tokens,branching", [(5, 10, (1, 1, 1)), (1, 5, (1,)), (6, 7, (2, 2))])
def test_finished_sequences_stay_inside_the_position_tables_cpu(time, new_tokens, branching):
    """Sequence 0 accepts a whole branch at every step, the others nothing, so it stands finished for
    many steps; ``max_seq_len`` is the least that is accepted. No node is ever past the tables, and
    the tokens are those of the same models with long tables."""
    tree, starts = TokenTree(branching), []
    branch = oracle.chains(tree.parents.tolist())[-1][::-1]

    def verify_tree(tokens, parents, p, u, q=None):
        batch = len(tokens)
        path = torch.full(tokens.shape, -1, dtype=torch.int32)
        path[:, 0] = 0
        path[0, :len(branch)] = torch.tensor(branch, dtype=torch.int32)
        counts = torch.ones(batch, dtype=torch.int32)
        counts[0] = len(branch)
        return path, counts, (tokens.sum(1) * 7 + 3) % SMALL.vocab_size

    def run(max_seq_len):
        config = DecoderConfig(vocab_size=96, dim=128, n_layers=1, n_heads=2, hidden_dim=128,
                               max_seq_len=max_seq_len)
        ops = _cpu_ops()
        attention = ops.tree_attention
        ops.tree_attention = lambda *a: (starts.append(int(a[-1].max())), attention(*a))[1]
        ops.verify_tree = verify_tree
        return generate_speculative(_model(3, config=config), _model(4, config=config),
                                    _prompt(3, time), new_tokens, branching, 1.0,
                                    torch.Generator().manual_seed(2), ops)[0]

    limit = time + new_tokens + len(branching)
    want = run(128)
    assert max(starts) + tree.depth < limit
    assert torch.equal(run(limit), want)
    with pytest.raises(ValueError, match="max_seq_len"):
        run(limit - 1)


def _without_finite_logits(config=SMALL):
    model = _model(3, config=config)
    with torch.no_grad():
        model.blocks[0].qkv.fill_(float("nan"))
    return model


def test_a_target_without_probabilities_raises_cpu():
    """All logits of the target are NaN: the walk draws no token (-1), and none may become a root."""
    with pytest.raises(RuntimeError, match="no token"):
        generate_speculative(_without_finite_logits(), _model(4), _prompt(2, 5), 6, (2, 1), 1.0,
                             torch.Generator().manual_seed(1), _cpu_ops())


@pytest.mark.parametrize("finished", [True, False])
def test_no_token_drawn_matters_to_running_sequences_only_cpu(finished):
    """Sequence 0 draws no token at the second step. That ends the call unless it needs none: it has
    finished before, or the accepted tokens are all that were asked for."""
    calls = []

    def verify_tree(tokens, parents, p, u, q=None):
        calls.append(None)
        batch, nodes = tokens.shape
        path = torch.arange(nodes, dtype=torch.int32).repeat(batch, 1)
        counts = torch.ones(batch, dtype=torch.int32)
        counts[0] = nodes
        nxt = torch.full((batch,), 5)
        if len(calls) >= 2:
            nxt[0] = -1
        return path, counts, nxt

    ops = _cpu_ops()
    ops.verify_tree = verify_tree
    # A chain of 3: sequence 0 has 4 tokens after a step, 8 after two.
    args = (_model(3), _model(4), _prompt(2, 5), 7 if finished else 8, (1, 1, 1), 1.0,
            torch.Generator().manual_seed(1), ops)
    if finished:
        out, _ = generate_speculative(*args)
        assert ((out >= 0) & (out < SMALL.vocab_size)).all() and len(calls) == 7
    else:
        with pytest.raises(RuntimeError, match="no token"):
            generate_speculative(*args)
        assert len(calls) == 2


def test_a_draft_without_probabilities_proposes_uniformly_cpu():
    """All logits of the draft are NaN: its tokens are drawn uniformly, which is what the walk is told,
    so the call goes on with the target's own tokens."""
    seen, ops = [], _cpu_ops()
    verify = ops.verify_tree
    ops.verify_tree = lambda *a: (seen.append(a[-1].clone()), verify(*a))[1]
    out, stats = generate_speculative(_model(3), _without_finite_logits(), _prompt(2, 5), 6, (2, 1), 1.0,
                                      torch.Generator().manual_seed(1), ops)
    assert ((out >= 0) & (out < SMALL.vocab_size)).all() and 1 <= stats["accepted"] <= 3
    inner = TokenTree((2, 1)).levels[-1][0]   # nodes with children
    assert all(torch.equal(q[:, :inner], torch.full_like(q[:, :inner], 1 / SMALL.vocab_size)) for q in seen)
