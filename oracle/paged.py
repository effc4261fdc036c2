"""Float64 restatement of the paged-cache operators and the norms around a
block (numpy; no device).  The 4-bit codes are restated in float32 with one
rounding per operation, as their definition has them, so that they compare
bit for bit."""
from __future__ import annotations

import numpy as np

from .reference import bf16_round


def rounder(dtype: str):
    """float32 -> float32 holding values of ``dtype``."""
    if dtype == "bfloat16":
        return lambda x: bf16_round(np.asarray(x, np.float32))
    if dtype == "float16":
        return lambda x: np.asarray(x, np.float32).astype(np.float16).astype(np.float32)
    return lambda x: np.asarray(x, np.float32)


def places(cu, used, table, tokens, block_size, pages, positions=None):
    """Per token: (sequence, position, page, row); sequence -1: left out, page
    -1: no cache row."""
    out = [(-1, 0, -1, 0)] * tokens
    for b in range(len(used)):
        b0, b1 = int(cu[b]), int(cu[b + 1])
        if b0 < 0 or b1 > tokens:
            continue
        for t in range(b0, b1):
            pos = int(used[b]) - (b1 - b0) + t - b0
            if pos < 0 or (positions is not None and pos >= positions):
                continue
            e = pos // block_size
            page = int(table[b, e]) if e < table.shape[1] else -1
            out[t] = (b, pos, page if 0 <= page < pages else -1, pos % block_size)
    return out


def rotate(x, cos, sin, interleaved, dtype=np.float64):
    """x [tokens, heads, d] by cos / sin [tokens, r / 2]; each operation rounds in ``dtype``."""
    x = x.astype(dtype)
    r = 2 * cos.shape[-1]
    c, s = cos.astype(dtype)[:, None], sin.astype(dtype)[:, None]
    y = x.copy()
    i0, i1 = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, b = x[..., i0], x[..., i1]
    y[..., i0] = a * c - b * s
    y[..., i1] = b * c + a * s
    return y


def quantize(x, dtype: str):
    """float32 rows x [..., d] -> codes uint8 [..., d], scale, offset [..., 1] (values of ``dtype``)."""
    rnd, f = rounder(dtype), np.float32
    x = x.astype(f)
    with np.errstate(all="ignore"):
        lo, hi = x.min(-1, keepdims=True), x.max(-1, keepdims=True)
        spread = hi - lo
        bad = ~np.isfinite(spread)
        s = rnd(spread / f(15))
        s = np.where(s < f(2.0 ** -126), f(0), s)
        o = rnd(lo + f(8) * s)
        inv = np.where(s > 0, f(1) / np.where(s > 0, s, f(1)), f(0)).astype(f)
        c = np.clip(np.rint((x - o) * inv) + f(8), 0, 15)
    c = np.where(bad, 0, c).astype(np.uint8)
    nan = f(np.nan)
    return c, np.where(bad, nan, s).astype(f), np.where(bad, nan, o).astype(f)


def pack(c):
    return (c[..., 0::2] | (c[..., 1::2] << 4)).astype(np.uint8)


def unpack(b):
    return np.stack([b & 15, b >> 4], -1).reshape(*b.shape[:-1], 2 * b.shape[-1])


def values(codes, scale):
    """float64 values of packed codes [..., d / 2] and scale pairs [..., 2]."""
    return (unpack(codes).astype(np.float64) - 8) * scale[..., :1].astype(np.float64) + scale[..., 1:].astype(np.float64)


def attention(q, k, v, used, cu, scale, left, right, seqlen_q, seen=None):
    """q [T, H, D]; k, v: per sequence [keys, HK, D] float64; seen: per sequence
    [keys] bool (a held page).  Returns o, lse [H, T] and the rows written."""
    t, h, d = q.shape
    o = np.zeros((t, h, d))
    lse = np.full((h, t), np.inf)
    rows = np.zeros(t, bool)
    for b in range(len(used)):
        b0, b1 = int(cu[b]), int(cu[b + 1])
        if b0 < 0 or b1 > t:
            continue
        n, keys = b1 - b0, k[b].shape[0]
        hk = k[b].shape[1]
        j = np.arange(keys)
        for i in range(min(n, seqlen_q)):
            rows[b0 + i] = True
            at = i + int(used[b]) - n
            vis = np.ones(keys, bool) if seen is None else seen[b].copy()
            if left >= 0:
                vis &= j >= at - left
            if right >= 0:
                vis &= j <= at + right
            if not vis.any():
                continue
            for hh in range(h):
                c = hh // (h // hk)
                s = (k[b][vis, c] @ q[b0 + i, hh].astype(np.float64)) * scale
                m = s.max()
                p = np.exp(s - m)
                o[b0 + i, hh] = p @ v[b][vis, c] / p.sum()
                lse[hh, b0 + i] = m + np.log(p.sum())
    return o, lse, rows


def block_norm(x, h, w_pre, eps, w_post=None, gate=None, act="none", alpha=1.0):
    x, u = x.astype(np.float64), h.astype(np.float64)
    if w_post is not None:
        u = u / np.sqrt((u * u).mean(-1, keepdims=True) + eps) * w_post.astype(np.float64)
    if gate is not None:
        g = gate.astype(np.float64)
        with np.errstate(over="ignore"):
            u = u * {"none": lambda z: z, "sigmoid": lambda z: 1 / (1 + np.exp(-z)), "tanh": np.tanh}[act](g)
    y = alpha * x + u
    n = None if w_pre is None else y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * w_pre.astype(np.float64)
    return y, n
