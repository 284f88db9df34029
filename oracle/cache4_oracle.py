"""64-bit restatement of the query/key norm and of the 4-bit KV cache (numpy; test infrastructure only).

Written from the definitions: nearest-value searches over the tables, one row or one query at a time.
"""
import numpy as np

MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
# Scale bytes 0 .. 0xE2: 5 bits of exponent (bias 15), 3 of mantissa, subnormals below 2^-14.
SCALES = np.array([(b % 8) * 2.0 ** -17 if b < 8 else (1 + b % 8 / 8) * 2.0 ** (b // 8 - 15)
                   for b in range(0xE3)])


def nearest(y, table):
    """Index of the nearest entry of an ascending table, of two the even one; saturating."""
    hi = np.clip(np.searchsorted(table, y), 1, len(table) - 1)
    lo = hi - 1
    down, up = y - table[lo], table[hi] - y
    even = np.where(lo % 2 == 0, lo, hi)
    return np.where(down < up, lo, np.where(up < down, hi, even))


def quantise(x):
    """Rows [..., 64] to (codes with their sign in bit 3 [..., 64], scale bytes [..., 4])."""
    g = np.asarray(x, np.float64).reshape(*x.shape[:-1], 4, 16)
    with np.errstate(all="ignore"):
        top = np.abs(g).max(-1)
        byte = nearest(np.where(np.isnan(top), 0.0, np.minimum(top / 6, SCALES[-1])), SCALES)
        scale = SCALES[byte][..., None]
        code = nearest(np.minimum(np.abs(g) / np.where(scale > 0, scale, 1.0), 6.0), MAGNITUDES)
    code = np.where(scale > 0, code, 0) + 8 * np.signbit(g)
    return code.reshape(x.shape), np.where(np.isnan(top), 0xFF, byte).astype(np.uint8)


def values(codes, scales):
    """What codes [..., 64] and scale bytes [..., 4] stand for."""
    scale = np.append(SCALES, np.full(256 - len(SCALES), np.nan))[scales]
    v = np.where(codes >= 8, -1.0, 1.0) * MAGNITUDES[codes % 8]
    return v * np.repeat(scale, 16, axis=-1)


def unpack(cache):
    """[B, H, n, 576] bytes to codes [B, H, 16 n, 64] and scale bytes [B, H, 16 n, 4]."""
    B, H, n, _ = cache.shape
    rows = cache[..., :512].reshape(B, H, n * 16, 32)
    codes = np.stack((rows & 15, rows >> 4), -1).reshape(B, H, n * 16, 64)
    return codes, cache[..., 512:].reshape(B, H, n * 16, 4)


def pack(codes, scales):
    """The reverse: codes [B, H, 16 n, 64] and scale bytes [B, H, 16 n, 4] to [B, H, n, 576] bytes."""
    B, H, rows, _ = codes.shape
    pairs = (codes[..., 0::2] + 16 * codes[..., 1::2]).astype(np.uint8)
    return np.concatenate((pairs.reshape(B, H, rows // 16, 512),
                           scales.astype(np.uint8).reshape(B, H, rows // 16, 64)), -1)


def norm_rope(x, w, cos, sin, eps):
    """Heads x [B, T, h, 64] normed by w (None: not) and turned by cos/sin [B or 1, T, 32]; also the sum of
    the magnitudes of each element's two terms."""
    x = np.asarray(x, np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    c, s = cos[:, :, None], sin[:, :, None]
    e, o = x[..., 0::2], x[..., 1::2]
    y = np.stack((e * c - o * s, e * s + o * c), -1).reshape(x.shape)
    mag = np.stack((abs(e * c) + abs(o * s), abs(e * s) + abs(o * c)), -1).reshape(x.shape)
    return y, mag


def norm_rope_backward(x, w, cos, sin, eps, g):
    """dx, dw (None without w) for gradients g [B, T, h, 64] of norm_rope's output, and the sums of magnitudes
    that bound their rounding errors."""
    c, s = cos[:, :, None], sin[:, :, None]
    e, o = g[..., 0::2], g[..., 1::2]
    n = np.stack((e * c + o * s, o * c - e * s), -1).reshape(g.shape)
    mag = np.stack((abs(e * c) + abs(o * s), abs(o * c) + abs(e * s)), -1).reshape(g.shape)
    if w is None:
        return n, None, mag, None
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    unit = x * r
    dw = (n * unit).sum((0, 1, 2))
    dx = r * (n * w - unit * (n * w * unit).mean(-1, keepdims=True))
    bound = r * (mag * abs(w) + abs(unit) * (mag * abs(w * unit)).mean(-1, keepdims=True))
    return dx, dw, bound, (mag * abs(unit)).sum((0, 1, 2))


def attention(q, k, v, lens):
    """Queries q [B, Hq, T, 64] over rows k, v [B, Hkv, C, 64]; query t sees j < lens[b] - (T - 1 - t). Returns O,
    LSE and the same average of |v|."""
    B, Hq, T, D = q.shape
    Hkv, C = k.shape[1], k.shape[2]
    o, a = np.zeros_like(q), np.zeros_like(q)
    lse = np.full((B, Hq, T), -np.inf)
    for b in range(B):
        for h in range(Hq):
            for t in range(T):
                n = min(max(int(lens[b]), 0), C) - (T - 1 - t)
                if n <= 0:
                    continue
                kv = h // (Hq // Hkv)
                s = k[b, kv, :n] @ q[b, h, t] / np.sqrt(D)
                m = s.max()
                p = np.exp(s - m)
                lse[b, h, t] = m + np.log(p.sum())
                o[b, h, t] = p @ v[b, kv, :n] / p.sum()
                a[b, h, t] = p @ np.abs(v[b, kv, :n]) / p.sum()
    return o, lse, a
