"""Timed cases of the 4-bit KV cache and of the query/key norm, with their plain forms.

The operators are reached through ``tiny_transformer_b200.operators``:

* ``fused.qkv_norm_rope``: RMS norm of every query and key head and the position rotation, in one
  pass over a fused QKV projection, with its gradients;
* ``cache4.append`` / ``cache4.read``: the same pass in front of a cache held in 4 bits, whose rows it
  quantises as it writes them, and the way back to BF16;
* ``cache4.attention`` / ``cache4.attention_with_lse``: attention of 1 to 16 query tokens over such a
  cache, with shared K/V heads and a length for each sequence.

A cache is uint8 ``[B, Hkv, ceil(C / 16), 576]``: blocks of 16 rows, 16 x 32 bytes of e2m1 codes (element
2i of a row in the low half of byte i) and 16 x 4 scales, one for 16 elements. A scale is the upper byte of
a half without its sign; a value is its code times its scale.

With ``own`` false, ``run`` computes the same with elementary torch operations. ``exact`` computes it once
more, in 64 bits, from the definitions.
"""
import math

import torch

own = False

HEAD_DIM = 64
EPS = 1e-6
THETA = 10000.0
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)       # e2m1 magnitudes
BORDERS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)       # between them; ties go to the even code
LARGEST_SCALE = 10240.0                                 # six times it is still finite in half precision

# ------------------------------------------------------------------------------- the cases


def listed():
    def norm(name, B, T, Hq, Hkv, positions, w32=False):
        return dict(name=name, op="norm", B=B, T=T, Hq=Hq, Hkv=Hkv, positions=positions, w32=w32)

    def append(name, B, T, Hq, Hkv, C, start, positions, normed):
        return dict(name=name, op="append", B=B, T=T, Hq=Hq, Hkv=Hkv, C=C, start=start,
                    positions=positions, normed=normed)

    def attn(name, B, T, Hq, Hkv, C, lo, hi, lse=False):
        return dict(name=name, op="attn", B=B, T=T, Hq=Hq, Hkv=Hkv, C=C, lo=lo, hi=hi, lse=lse)

    return [
        # Training on one short sequence of the framework's decoder: latency.
        norm("norm_b1_t128_h12", 1, 128, 12, 12, "int"),
        # Shared K/V heads, an odd length, packed documents (a position for every token), FP32 weights.
        norm("norm_b3_t1021_h12_kv4", 3, 1021, 12, 4, "every", w32=True),
        # The training shape of the framework's attention benchmark.
        norm("norm_b4_t4096_h12", 4, 4096, 12, 12, "int"),
        # A decode step of one user: the position is on the device, as in a captured step.
        append("append_b1_t1_c512", 1, 1, 12, 12, 512, 300, "one", False),
        # A decode step of the large serving batch, every sequence at a position of its own.
        append("append_b64_t1_c8192", 64, 1, 12, 12, 8192, 5000, "each", True),
        # A chunk of a prompt behind an odd prefix, shared K/V heads; the prefix is read back with it.
        append("append_b3_t1021_h12_kv4", 3, 1021, 12, 4, 2048, 37, "int", True),
        # A large batch of prompts, written and read back for the prompt's own attention.
        append("append_b4_t4096_h12", 4, 4096, 12, 12, 4096, 0, "int", True),
        # One user over a short cache: latency.
        attn("attn_b1_c512", 1, 1, 12, 12, 512, 300, 512),
        # A few new tokens of each sequence, shared K/V heads, odd sizes, LSE too.
        attn("attn_b3_t5_h12_kv4_c20001", 3, 5, 12, 4, 20001, 9000, 20001, lse=True),
        # A serving batch with shared K/V heads over caches of the decoder's longest length.
        attn("attn_b32_h32_kv8_c4096", 32, 1, 32, 8, 4096, 1024, 4096),
        # The large serving batch of the decode benchmark, cache lengths 1024 to 8192.
        attn("attn_b64_h12_c8192", 64, 1, 12, 12, 8192, 1024, 8192),
        # One user's long context, few K/V heads.
        attn("attn_b1_h16_kv2_c131072", 1, 1, 16, 2, 131072, 130000, 131072),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(12, 12), (12, 12), (8, 8), (12, 4), (8, 2), (6, 3), (16, 2), (32, 8), (9, 1)]


def draw(rng):
    op = rng.choice(["norm", "append", "append", "attn", "attn", "attn"])
    Hq, Hkv = rng.choice(HEADS)
    if op == "attn":
        B, C = _log_int(rng, 1, 64), _log_int(rng, 64, 131072)
        T = rng.choice([1, 1, 1, 1, rng.randint(2, 16)])
        while B > 1 and (B * Hkv * C > 64 * 12 * 4608 or B * Hq * T * C > 64 * 12 * 8192):
            B = B // 2
        hi = rng.randint(C // 2, C)
        return dict(op=op, B=B, T=T, Hq=Hq, Hkv=Hkv, C=C, lo=rng.randint(0, hi), hi=hi,
                    lse=rng.random() < 0.5)
    B, T = _log_int(rng, 1, 64), rng.choice([1, _log_int(rng, 1, 4096), _log_int(rng, 1, 4096)])
    while B > 1 and B * T * (Hq + 2 * Hkv) > 4 * 4096 * 36:
        B = B // 2
    if op == "norm":
        return dict(op=op, B=B, T=T, Hq=Hq, Hkv=Hkv, w32=rng.random() < 0.3,
                    positions=rng.choice(["int", "each", "every"]))
    positions = rng.choice(["int", "one", "each"])
    # A prompt's prefix comes back whole: no more rows than the largest listed case has.
    last = 8192 if positions != "int" else min(8192, max(T, 4 * 12 * 4096 // (B * Hkv)))
    start = rng.randint(0, last - T)
    return dict(op=op, B=B, T=T, Hq=Hq, Hkv=Hkv, C=rng.randint(start + T, 8192), start=start,
                positions=positions, normed=rng.random() < 0.7)


# ------------------------------------------------------------------------------- inputs


def _lengths(case):
    """B lengths spread evenly over [lo, hi]: the same multiset for every seed."""
    B, lo, hi = case["B"], case["lo"], case["hi"]
    return [lo + int((hi - lo) * (i + 0.5) / B) for i in range(B)]


def _starts(case):
    """First positions of the B sequences: different ones where each sequence has its own."""
    B, start = case["B"], case["start"]
    if case["positions"] != "each":
        return [start] * B
    return [int(start * (i + 1) / B) for i in range(B)]


def _prefix(case):
    """Rows that come back from one pass of the append: a prompt's whole prefix, a step's own rows."""
    return case["start"] + case["T"] if case["positions"] == "int" else case["T"]


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _filled_cache(gen, B, H, C):
    """A cache whose rows hold normal values, made sequence by sequence."""
    blocks = (C + 15) // 16
    out = torch.zeros(B, H, blocks, 576, device="cuda", dtype=torch.uint8)
    for b in range(B):
        _encode_rows(out[b:b + 1], 0, _randn(gen, 1, H, blocks * 16, HEAD_DIM).to(torch.bfloat16))
    return out


def _tables(positions):
    freq = 1.0 / THETA ** (torch.arange(0, HEAD_DIM, 2, device="cuda").double() / HEAD_DIM)
    angles = torch.arange(positions, device="cuda").double()[:, None] * freq
    return angles.cos().float(), angles.sin().float()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, T, Hq, Hkv = case["B"], case["T"], case["Hq"], case["Hkv"]
    s = dict(op=case["op"], Hq=Hq, Hkv=Hkv)
    if case["op"] == "attn":
        C = case["C"]
        # Queries as they leave the fused projection of a step: a transposed view.
        s["q"] = _randn(gen, B, T, Hq, HEAD_DIM).to(torch.bfloat16).transpose(1, 2)
        s["cache_k"], s["cache_v"] = _filled_cache(gen, B, Hkv, C), _filled_cache(gen, B, Hkv, C)
        order = torch.randperm(B, generator=gen, device="cuda")
        s["kv_lens"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")[order]
        s["lse"] = case["lse"]
        return s
    # Projections of a decoder whose features differ in size, with a few large ones.
    size = torch.exp(0.5 * _randn(gen, Hq + 2 * Hkv, HEAD_DIM))
    s["qkv"] = (_randn(gen, B, T, Hq + 2 * Hkv, HEAD_DIM) * size).to(torch.bfloat16)
    w = [1.0 + 0.2 * _randn(gen, HEAD_DIM) for _ in range(2)]
    if not case.get("w32"):
        w = [x.to(torch.bfloat16) for x in w]
    s["q_weight"], s["k_weight"] = w
    if case["op"] == "norm":
        s["cos"], s["sin"] = _tables(max(8192, T))
        s["position"] = 0
        if case["positions"] == "each":
            s["position"] = torch.randint(0, 8192 - T + 1, (B,), generator=gen, device="cuda")
        elif case["positions"] == "every":    # documents packed into a row: positions start again
            at = torch.arange(T, device="cuda")
            cut = torch.randint(0, T, (B, 1), generator=gen, device="cuda")
            s["position"] = torch.where(at < cut, at, at - cut).contiguous()
        s["grads"] = [_randn(gen, B, h, T, HEAD_DIM).to(torch.bfloat16) for h in (Hq, Hkv, Hkv)]
        for x in ("qkv", "q_weight", "k_weight"):
            s[x].requires_grad_()
        return s
    s["cos"], s["sin"] = _tables(8192)
    if not case["normed"]:
        s["q_weight"] = s["k_weight"] = None
    starts = _starts(case)
    s["position"] = starts[0]
    if case["positions"] == "one":
        s["position"] = torch.tensor(starts[:1], device="cuda")
    elif case["positions"] == "each":
        order = torch.randperm(B, generator=gen, device="cuda")
        s["position"] = torch.tensor(starts, device="cuda")[order]
    s["from"], s["rows"] = (0 if case["positions"] == "int" else s["position"]), _prefix(case)
    s["cache_k"], s["cache_v"] = (_filled_cache(gen, B, Hkv, case["C"]) for _ in range(2))
    return s


# ------------------------------------------------------------------------------- one pass


def run(state):
    s = state
    if own:
        from __graft_entry__ import import_package
        import_package()
        from tiny_transformer_b200.operators import cache4, fused
        if s["op"] == "norm":
            leaves = (s["qkv"], s["q_weight"], s["k_weight"])
            q, k, v = fused.qkv_norm_rope(*leaves, s["cos"], s["sin"], s["position"], eps=EPS,
                                          kv_heads=s["Hkv"])
            return [q, k, v, *torch.autograd.grad((q, k, v), leaves, s["grads"])]
        if s["op"] == "append":
            q = cache4.append(s["qkv"], s["cos"], s["sin"], s["position"], s["cache_k"], s["cache_v"],
                              s["q_weight"], s["k_weight"], eps=EPS)
            return [q, *cache4.read(s["cache_k"], s["cache_v"], s["from"], s["rows"])]
        call = cache4.attention_with_lse if s["lse"] else cache4.attention
        return call(s["q"], s["cache_k"], s["cache_v"], s["kv_lens"])
    with torch.no_grad():
        if s["op"] == "norm":
            return _plain_norm(s)
        return _plain_append(s) if s["op"] == "append" else _plain_attention(s)


def _angles(s, B, T):
    """cos and sin of every token, [B or 1, T, 1, 32]."""
    p = s["position"]
    if not torch.is_tensor(p):
        p = torch.tensor([p], device=s["cos"].device)
    if p.dim() == 1:
        p = p[:, None] + torch.arange(T, device=p.device)
    return s["cos"][p][:, :, None], s["sin"][p][:, :, None]


def _rotate(x, c, s):
    even, odd = x[..., 0::2], x[..., 1::2]
    return torch.stack((even * c - odd * s, even * s + odd * c), -1).flatten(-2)


def _plain_norm(s):
    Hq, Hkv = s["Hq"], s["Hkv"]
    B, T = s["qkv"].shape[:2]
    c, sn = _angles(s, B, T)
    parts = s["qkv"].split([Hq, Hkv, Hkv], 2)
    out, dx, dw = [], [], []
    for x, w, g in zip(parts, (s["q_weight"], s["k_weight"]), s["grads"]):
        x, wf, g = x.float(), w.float(), g.float().transpose(1, 2)
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
        n = x * r
        out.append(_rotate(n * wf, c, sn).to(torch.bfloat16).transpose(1, 2))
        g = _rotate(g, c, -sn)
        dw.append((g * n).double().sum((0, 1, 2)).to(w.dtype))
        g = g * wf
        dx.append(((g - n * (g * n).mean(-1, keepdim=True)) * r).to(torch.bfloat16))
    dx.append(s["grads"][2].transpose(1, 2))
    return [*out, parts[2].transpose(1, 2), torch.cat(dx, 2), *dw]


def _encode_rows(cache, start, x):
    """Quantise the BF16 rows x [B, H, T, 64] into rows start + t of a cache (start: an int or [B])."""
    B, H, T, _ = x.shape
    g = x.double().view(B, H, T, 4, 16)
    size = g.abs()
    want = size.amax(-1, keepdim=True) / 6
    # Four significant bits, to even; below 2^-14 the fixed steps of a half's upper byte.
    step = torch.exp2(torch.frexp(want)[1].double().clamp(min=-13) - 4)
    scale = (torch.round(want / step) * step).clamp(max=LARGEST_SCALE)
    byte = scale.half().view(torch.int16).bitwise_right_shift(7).to(torch.uint8)
    code = torch.zeros(B, H, T, 4, 16, dtype=torch.uint8, device=x.device)
    for i, border in enumerate(BORDERS):
        code += (size > border * scale) if i % 2 == 0 else (size >= border * scale)
    code = torch.where(scale > 0, code, 0) + 8 * torch.signbit(g).to(torch.uint8)
    pairs = code.view(B, H, T, 32, 2)
    pairs = pairs[..., 0] + 16 * pairs[..., 1]
    at = torch.as_tensor(start, device=x.device).reshape(-1, 1) + torch.arange(T, device=x.device)
    b = torch.arange(B, device=x.device)[:, None]
    codes, scales = _parts(cache)
    codes[b, :, at // 16, at % 16] = pairs.transpose(1, 2)
    scales[b, :, at // 16, at % 16] = byte[..., 0].transpose(1, 2)


def _parts(cache):
    B, H, n, _ = cache.shape
    return (cache[..., :512].unflatten(-1, (16, 32)), cache[..., 512:].unflatten(-1, (16, 4)))


def _decode_rows(cache):
    """Every row of a cache in FP32, [B, H, 16 n, 64]."""
    codes, scales = _parts(cache)
    B, H, n = codes.shape[:3]
    codes = torch.stack((codes & 15, codes >> 4), -1).view(B, H, n * 16, 4, 16)
    signed = torch.tensor(VALUES + tuple(-x for x in VALUES), device=cache.device)
    scale = scales.to(torch.int16).bitwise_left_shift(7).view(torch.float16).float()
    return (signed[codes.int()] * scale.reshape(B, H, n * 16, 4, 1)).view(B, H, n * 16, HEAD_DIM)


def _plain_append(s):
    Hq, Hkv = s["Hq"], s["Hkv"]
    B, T = s["qkv"].shape[:2]
    c, sn = _angles(s, B, T)
    q, k, v = s["qkv"].split([Hq, Hkv, Hkv], 2)
    # The keys in 64 bits: an error of the last bit, next to a border, is a whole step of a code.
    q, k, ck, sk = q.float(), k.double(), c.double(), sn.double()
    if s["q_weight"] is not None:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * s["q_weight"].float()
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * s["k_weight"].double()
    q = _rotate(q, c, sn).to(torch.bfloat16).transpose(1, 2)
    k = _rotate(k, ck, sk).to(torch.bfloat16).transpose(1, 2)
    start = s["position"]
    _encode_rows(s["cache_k"], start, k)
    _encode_rows(s["cache_v"], start, v.transpose(1, 2))
    at = torch.as_tensor(s["from"], device=q.device).reshape(-1, 1) + torch.arange(s["rows"], device=q.device)
    at = at.expand(B, -1)
    b = torch.arange(B, device=q.device)[:, None]
    rows = []
    for cache in (s["cache_k"], s["cache_v"]):
        if s["rows"] <= 16:      # a step: its own blocks alone
            touched = _decode_rows(cache[b, :, at // 16].transpose(1, 2))
            touched = touched.unflatten(2, (s["rows"], 16))
            i = torch.arange(s["rows"], device=q.device)[None]
            rows.append(touched[b, :, i, at % 16].transpose(1, 2).to(torch.bfloat16))
        else:
            rows.append(_decode_rows(cache)[b, :, at].transpose(1, 2).to(torch.bfloat16))
    return [q, *rows]


def _plain_attention(s):
    q, lens = s["q"].float(), s["kv_lens"]
    B, Hq, T, _ = q.shape
    Hkv = s["Hkv"]
    k = _decode_rows(s["cache_k"])
    C = k.shape[2]
    # Query t of T sees all rows but the last T - 1 - t of its sequence.
    end = lens[:, None] - (T - 1) + torch.arange(T, device=q.device)
    mask = (torch.arange(C, device=q.device) < end[..., None])[:, None, None]       # [B, 1, 1, T, C]
    scores = torch.matmul(q.reshape(B, Hkv, -1, HEAD_DIM), k.transpose(2, 3)).mul_(0.125)
    del k
    scores = scores.view(B, Hkv, Hq // Hkv, T, C).masked_fill_(~mask, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top > float("-inf"), top, torch.zeros((), device=q.device))
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    seen = torch.arange(C, device=q.device) < lens[:, None]
    v = _decode_rows(s["cache_v"]).masked_fill_(~seen[:, None, :, None], 0.0)
    o = torch.matmul(p.view(B, Hkv, -1, C), v).view(B, Hkv, -1, T, HEAD_DIM)
    o = torch.where(total > 0, o / total, torch.zeros((), device=q.device))
    o = o.to(torch.bfloat16).reshape(B, Hq, T, HEAD_DIM)
    return (o, (top + total.log()).reshape(B, Hq, T)) if s["lse"] else o


# ------------------------------------------------------------------------------- 64 bits


def _exact_positions(s, B, T):
    p = s["position"]
    if not torch.is_tensor(p):
        p = torch.full((B,), p, device="cuda")
    if p.dim() == 2:
        return p
    return p.expand(B)[:, None] + torch.arange(T, device="cuda")


def _exact_turn(x, w, cos, sin):
    """Norm and rotation of [..., 64] heads, pairs as complex numbers; w None: the rotation alone."""
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    z = torch.view_as_complex(x.unflatten(-1, (32, 2)).contiguous()) * torch.complex(cos, sin)
    return torch.view_as_real(z).flatten(-2)


def _exact_quantised(x):
    """The values that 64-bit rows [..., 64] come back as: nearest code, of two the one with the even
    number, times a scale rounded in the same way."""
    g = x.unflatten(-1, (4, 16))
    most = g.abs().amax(-1, keepdim=True)
    grid = torch.arange(256, dtype=torch.int16, device=x.device).bitwise_left_shift(7)
    grid = grid.view(torch.float16).double()
    grid = grid[grid <= LARGEST_SCALE]

    def nearest(y, table):       # y >= 0; table ascending, ties to the entry with the even index
        hi = torch.searchsorted(table, y.contiguous()).clamp(1, len(table) - 1)
        lo = hi - 1
        down, up = y - table[lo], table[hi] - y
        even = torch.where(lo % 2 == 0, lo, hi)
        return table[torch.where(down < up, lo, torch.where(up < down, hi, even))]

    scale = nearest(most / 6, grid)
    table = torch.tensor(VALUES, dtype=torch.float64, device=x.device)
    safe = torch.where(scale > 0, scale, 1.0)
    code = nearest((g.abs() / safe).clamp(max=6.0), table) * torch.sign(g)
    return torch.where(scale > 0, code * scale, 0.0).flatten(-2)


def _exact_rows(cache, b, h):
    """Rows of one head of a cache in 64 bits."""
    codes = cache[b, h, :, :512].reshape(-1, 32).long()
    scales = cache[b, h, :, 512:].reshape(-1, 4).long()
    both = torch.stack((codes % 16, codes // 16), -1).flatten(1)
    kind = both % 8
    mag = torch.where(kind < 2, kind * 0.5, (1 + 0.5 * (kind % 2).double()) * 2.0 ** (kind // 2 - 1).double())
    exponent, fraction = scales // 8, (scales % 8).double()
    scale = torch.where(exponent == 0, fraction * 2.0 ** -17,
                        (1 + fraction / 8) * 2.0 ** (exponent - 15).double())
    return torch.where(both < 8, mag, -mag) * scale.repeat_interleave(16, 1)


def exact(case, seed):
    s = prepare(case, seed)
    B, T, Hq, Hkv = case["B"], case["T"], case["Hq"], case["Hkv"]
    if case["op"] == "attn":
        return _exact_attention(s, case)
    at = _exact_positions(s, B, T)
    cos, sin = (s[x].double()[at][:, :, None] for x in ("cos", "sin"))
    if case["op"] == "norm":
        leaves = [s[x].detach().double().requires_grad_() for x in ("qkv", "q_weight", "k_weight")]
        x = leaves[0]
        q = _exact_turn(x[:, :, :Hq], leaves[1], cos, sin).transpose(1, 2)
        k = _exact_turn(x[:, :, Hq:Hq + Hkv], leaves[2], cos, sin).transpose(1, 2)
        v = x[:, :, Hq + Hkv:].transpose(1, 2)
        grads = torch.autograd.grad((q, k, v), leaves, [g.double() for g in s["grads"]])
        return [q.detach(), k.detach(), v.detach(), *grads]
    x = s["qkv"].double()
    w = [None if s[n] is None else s[n].double() for n in ("q_weight", "k_weight")]
    q = _exact_turn(x[:, :, :Hq], w[0], cos, sin).transpose(1, 2)
    k = _exact_turn(x[:, :, Hq:Hq + Hkv], w[1], cos, sin)
    new = [_exact_quantised(r).transpose(1, 2)
           for r in (k.to(torch.bfloat16).double(), x[:, :, Hq + Hkv:])]
    if s["rows"] == T:
        return [q, *new]
    before = [torch.stack([torch.stack([_exact_rows(s[n], b, h)[:case["start"]] for h in range(Hkv)])
                           for b in range(B)]) for n in ("cache_k", "cache_v")]
    return [q, *(torch.cat(both, 2) for both in zip(before, new))]


def _exact_attention(s, case):
    B, T, Hq, Hkv = case["B"], case["T"], case["Hq"], case["Hkv"]
    G = Hq // Hkv
    o = torch.zeros(B, Hq, T, HEAD_DIM, dtype=torch.float64, device="cuda")
    lse = torch.full((B, Hq, T), float("-inf"), dtype=torch.float64, device="cuda")
    lens = s["kv_lens"].tolist()
    for b in range(B):
        for h in range(Hkv):
            heads = slice(h * G, (h + 1) * G)
            k, v = (_exact_rows(s[x], b, h) for x in ("cache_k", "cache_v"))
            scores = s["q"][b, heads].double() @ k.T / math.sqrt(HEAD_DIM)          # [G, T, C]
            for t in range(T):
                n = lens[b] - (T - 1 - t)
                if n > 0:
                    row = scores[:, t, :n]
                    lse[b, heads, t] = torch.logsumexp(row, -1)
                    o[b, heads, t] = torch.softmax(row, -1) @ v[:n]
    return (o, lse) if case["lse"] else o


# ------------------------------------------------------------------------------- least work


def work(case):
    """Each input that the pass needs read once, each output written once."""
    B, T, Hq, Hkv = case["B"], case["T"], case["Hq"], case["Hkv"]
    row = 2 * HEAD_DIM                       # bytes of a head of one token in BF16
    if case["op"] == "attn":
        rows = sum(_lengths(case))
        return dict(bytes=2 * 36 * Hkv * rows + 2 * row * B * Hq * T + 4 * B
                    + (4 * B * Hq * T if case["lse"] else 0),
                    flops=4 * HEAD_DIM * Hq * T * rows)
    turned, every = Hq + Hkv, Hq + 2 * Hkv
    tables = 2 * 4 * 32 * T * (B if case["positions"] in ("each", "every") else 1)
    if case["op"] == "norm":
        # The projection's queries and keys, their norms, three gradients, the projection's gradient.
        return dict(bytes=row * B * T * (2 * turned + 2 * every) + tables,
                    flops=30 * HEAD_DIM * B * T * turned)
    # The projection, the queries, the rows' codes and scales, and the prefix that comes back.
    kept = _prefix(case) - T
    return dict(bytes=B * T * (row * (every + Hq) + 72 * Hkv) + tables
                + B * Hkv * (72 * kept + 2 * row * (kept + T)),
                flops=B * T * HEAD_DIM * (12 * turned + 20 * Hkv))
