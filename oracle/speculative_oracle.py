"""CPU oracle of the speculative-decoding operators: plain restatements in 64 bits (numpy)."""
from __future__ import annotations

import math

import numpy as np

ONE = 1 << 36


def chains(parents):
    """For each node the list of itself and its ancestors; [] when the node is not in use."""
    out = []
    for n in range(len(parents)):
        chain, m = [], n
        while m >= 0:
            chain.append(m)
            up = int(parents[m])
            m = up if -1 <= up < m else -2
        out.append(chain if m == -1 else [])
    return out


def tree_attention(q, tree_k, tree_v, cache_k, cache_v, parents, lens):
    """(O, LSE, A) in float64; A is the same average of |v|, the scale of rounding errors in the
    weights. Inputs are float64 arrays [B, Hq, N, D], [B, Hkv, N, D], [B, Hkv, C, D]; parents [B, N]."""
    B, Hq, N, D = q.shape
    Hkv, C = cache_k.shape[1:3]
    O, A = np.zeros(q.shape), np.zeros(q.shape)
    lse = np.full((B, Hq, N), -np.inf)
    for b in range(B):
        L = min(max(int(lens[b]), 0), C)
        for n, chain in enumerate(chains(parents[b])):
            if not chain:
                continue
            for h in range(Hq):
                g = h // (Hq // Hkv)
                k = np.concatenate([cache_k[b, g, :L], tree_k[b, g, chain]])
                v = np.concatenate([cache_v[b, g, :L], tree_v[b, g, chain]])
                s = k @ q[b, h, n] / math.sqrt(D)
                top = s.max()
                w = np.exp(s - top)
                lse[b, h, n] = top + math.log(w.sum())
                w /= w.sum()
                O[b, h, n], A[b, h, n] = w @ v, w @ np.abs(v)
    return O, lse, A


def verify_tree(tokens, parents, p, u, q=None):
    """(path, counts, next) of the walk; whole numbers are Python integers."""
    B, N, V = p.shape
    path, counts = np.full((B, N), -1, np.int32), np.zeros(B, np.int32)
    nxt = np.full(B, -1, np.int64)
    for b in range(B):
        if parents[b, 0] != -1:
            continue
        cur, taken = 0, [0]
        while True:
            pc = np.clip(np.nan_to_num(p[b, cur], nan=0.0), 0, 1).astype(np.float64)
            base = np.floor(pc * ONE).astype(np.int64)
            r, S, hit = base.copy(), None, None
            for c in [c for c in range(cur + 1, N) if parents[b, c] == cur]:
                t = int(tokens[b, c])
                known = 0 <= t < V
                if q is None:
                    qc = np.zeros(V)
                    qc[t if known else slice(0, 0)] = 1.0
                    qt = 1.0
                else:
                    qc = np.clip(np.nan_to_num(q[b, cur], nan=0.0), 0, 1).astype(np.float64)
                    qt = qc[t] if known else 0.0
                if S is None:
                    ok = known and np.float32(u[b, c]) * np.float32(qt) < np.float32(pc[t])
                else:
                    ok = known and float(u[b, c]) * float(qt) * float(S) < float(r[t])
                if ok:
                    hit = c
                    break
                r = np.maximum(r - np.floor(qc * float(ONE if S is None else S)).astype(np.int64), 0)
                S = int(r.sum())
            if hit is None:
                break
            cur = hit
            taken.append(cur)
        if r.sum() == 0:
            r = base
        total = int(r.sum())
        if total > 0:
            goal = math.floor(float(u[b, 0]) * float(total))
            nxt[b] = int(np.searchsorted(np.cumsum(r), goal, side="right"))
        path[b, :len(taken)], counts[b] = taken, len(taken)
    return path, counts, nxt
