"""Plain restatements of the quantized cache and the attention over it: blocks
in numpy f32 steps, attention in 64 bits, one query at a time."""
from __future__ import annotations

import numpy as np

Q4_0, Q8_0 = 2, 8


def quantize(x, qtype):
    """int values and f16 scales of the blocks of f32 x [..., dim]."""
    b = np.asarray(x, np.float32).reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    with np.errstate(all="ignore"):
        if qtype == Q8_0:
            d = np.abs(b).max(-1) / np.float32(127)
        else:
            hi, lo = b.max(-1), b.min(-1)
            d = np.where(hi >= -lo, hi, lo) / np.float32(-8)
        d = np.where(np.isnan(b).any(-1), np.float32(np.nan), d).astype(np.float16)
        f = d.astype(np.float32)
        r = np.where(f != 0, np.float32(1) / np.where(f != 0, f, np.float32(1)), np.float32(0)).astype(np.float32)
        q = np.rint(b * r[..., None])
        q = np.clip(np.where(np.isnan(q), 0, q), *((-127, 127) if qtype == Q8_0 else (-8, 7)))
    return q, d


def values(x, qtype):
    """What the blocks of x stand for (f64; exact in f32)."""
    q, d = quantize(x, qtype)
    with np.errstate(invalid="ignore"):
        return (q.astype(np.float64) * d.astype(np.float64)[..., None]).reshape(x.shape)


def row_position(j, n, length, tree=None):
    return length - n + (int(tree[j].sum()) - 1 if tree is not None else j)


def visible(j, n, length, *, causal=True, window=0, prefix=0, first=0, tree=None):
    """Which of `length` keys query j of n sees; tree: [n, n] truth values."""
    keys = np.arange(length)
    base = length - n
    pos = row_position(j, n, length, tree)
    at = keys.copy()
    if tree is None:
        see = (keys <= pos) | (keys < prefix) if causal else np.ones(length, bool)
    else:
        see = keys < base
        for i in range(n):
            if 0 <= base + i < length:
                at[base + i] = row_position(i, n, length, tree)
                see[base + i] = tree[j, i]
    if first:
        see &= (keys >= first) | (keys >= base if tree is not None else False)
    if window:
        see &= np.abs(pos - at) < window
    return see, pos, at


def attend(q, k, v, starts, lens, *, scale=0.0, softcap=0.0, slopes=None, first=None, prefix=None, trees=None, **mask):
    """q [tokens, heads, dim]; k, v: a list per sequence of [len, kv heads, dim]
    values. The result in 64 bits and how far an f32 evaluation may be from it:
    a score is off by what its products and its size round to, a weight by that,
    the result by twice that of the largest value seen."""
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    T, Hq, D = q.shape
    scale = scale or D ** -0.5
    for s in range(len(lens)):
        n, L = int(starts[s + 1] - starts[s]), int(lens[s])
        if L == 0:
            continue
        G = Hq // k[s].shape[1]
        for j in range(n):
            t = int(starts[s]) + j
            see, pos, at = visible(j, n, L, prefix=0 if prefix is None else int(prefix[s]),
                                   first=0 if first is None else int(first[t]), tree=None if trees is None else trees[s], **mask)
            if not see.any():
                continue
            for h in range(Hq):
                kk, vv = k[s][see, h // G], v[s][see, h // G]
                with np.errstate(invalid="ignore", over="ignore"):
                    x = kk @ q[t, h].astype(np.float64) * scale
                    size = (np.abs(kk) @ np.abs(q[t, h]).astype(np.float64) * abs(scale)).max()
                    if softcap:
                        x, size = softcap * np.tanh(x / softcap), size + softcap
                    if slopes is not None:
                        far = np.abs(pos - at[see]) * float(slopes[h])
                        x, size = x - far, size + np.abs(far).max()
                    p = np.exp(x - x.max())
                    out[t, h] = p @ vv / p.sum()
                    tol[t, h] = np.abs(vv).max() * (2 * size * 2.0 ** -21 + 2.0 ** -20 + np.sqrt(see.sum()) * 2.0 ** -23) + 1e-30
    return out, tol
