"""Norms around a block in float64 with the error that each output may have.

u = 2^-24, half a step of fp32.  A row's squares are summed by threads of at most 32 or
cols / 256 elements, then over 64 lanes and 16 waves: all terms positive, so the sum is off by
k = max(32, cols / 256) + 22 u of itself, its inverse root by half that and 4 u (mean, eps,
root, division).  The block's term H r W_post act(G): two products, three with a gate; the
gate's exp takes an argument rounded to u of itself, |g| u of the result (2 |g| in tanh), and
its quotient at most 20 u more (near 0.18, where 1 - e^-2|g| cancels; the series below it
leaves out 2.5e-8 of g).  Y's sum: u of Y.  N: Y's own error, half of what it does to the sum of
squares, that sum's, two products.  Each output rounds once to its type.
"""
import numpy as np

from oracle import paged as ref

u = 2.0 ** -24
HALF = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 2.0 ** -149, "bfloat16": 2.0 ** -133, "float16": 2.0 ** -24}


def bounds(i, dt, act="none", alpha=1.0, eps=1e-6):
    """y, n and how far each may be off."""
    y, n = ref.block_norm(i["x"], i["h"], i["w_pre"], eps, i["w_post"], i["gate"], act, alpha)
    term = np.abs(y - alpha * i["x"].astype(np.float64))
    k = max(32, y.shape[1] / 256) + 22
    rel = 1.0
    if i["w_post"] is not None:
        rel += k / 2 + 4 + 2
    if i["gate"] is not None:
        rel = rel + 1 + (0 if act == "none" else 20 + 2 * np.abs(i["gate"].astype(np.float64)))
    dy = u * (rel * term + np.abs(y))
    by = dy + HALF[dt] * (np.abs(y) + dy) + TINY[dt]
    if n is None:
        return y, n, by, None
    ss = (y * y).sum(-1, keepdims=True)
    root = np.sqrt(ss / y.shape[1] + eps)
    ds = (np.abs(y) * dy).sum(-1, keepdims=True) / ss.clip(1e-300)
    dn = np.abs(n) * (ds + u * (k / 2 + 4 + 2)) + dy / root * np.abs(i["w_pre"].astype(np.float64))
    return y, n, by, dn + HALF[dt] * (np.abs(n) + dn) + TINY[dt]


def check(want, y, n):
    """y, n (float64 arrays) of a call against ``bounds``'s."""
    for got, w, bar in ((y, want[0], want[2]), (n, want[1], want[3])):
        if w is None:
            assert got is None
            continue
        off = np.abs(got - w) / bar
        assert (off <= 1).all(), float(np.nanmax(off))
