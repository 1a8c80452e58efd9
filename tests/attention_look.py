"""Attention over a cache in 64 bits with a tolerance for each block of 32 dims
by itself, for keys bounded by `most` and trees whose drafts may have no key."""
from __future__ import annotations

import numpy as np

from tests import attention_oracle as A


def attend(q, k, v, starts, lens, *, scale=0.0, softcap=0.0, slopes=None, first=None, prefix=None, trees=None, most=None, **mask):
    """As attention_oracle.attend. The tolerance of a result: what the scores
    round to (2^-21 of the terms' sum, twice: numerator and sum of weights),
    2^-20 for the weights' and values' two f16 terms, and 2^-23 for each of n
    sums taken at random, of the largest value seen in the same block."""
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    T, Hq, D = q.shape
    scale = scale or D ** -0.5
    for s in range(len(lens)):
        n, L = int(starts[s + 1] - starts[s]), int(lens[s])
        G = Hq // k[s].shape[1]
        for j in range(n):
            t = int(starts[s]) + j
            see, pos, at = A.visible(j, n, L, prefix=0 if prefix is None else int(prefix[s]),
                                     first=0 if first is None else int(first[t]), tree=None if trees is None else trees[s], **mask)
            if most is not None:
                see &= np.arange(L) < most
            if not see.any():
                continue
            for h in range(Hq):
                kk, vv = k[s][see, h // G], v[s][see, h // G]
                x = kk @ q[t, h].astype(np.float64) * scale
                size = (np.abs(kk) @ np.abs(q[t, h]).astype(np.float64) * abs(scale)).max()
                if softcap:
                    x, size = softcap * np.tanh(x / softcap), min(size, size + softcap)
                if slopes is not None:
                    far = np.abs(pos - at[see]) * float(slopes[h])
                    x, size = x - far, size + np.abs(far).max()
                p = np.exp(x - x.max())
                out[t, h] = p @ vv / p.sum()
                top = np.repeat(np.abs(vv).max(0).reshape(-1, 32).max(-1), 32)
                tol[t, h] = top * (2 * size * 2.0 ** -21 + 2.0 ** -20 + np.sqrt(see.sum()) * 2.0 ** -23) + 1e-30
    return out, tol
