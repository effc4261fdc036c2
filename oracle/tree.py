"""Float64 restatement of the operators on drafted trees (numpy; no device):
rows and positions of a tree's tokens, attention of its nodes, verification and
the move of the accepted rows."""
from __future__ import annotations

import numpy as np


def bounds(cu, used, tokens, z):
    """First row, nodes and base (keys before the tree) of sequence z."""
    b0, b1 = int(cu[z]), int(cu[z + 1])
    n = b1 - b0 if b0 >= 0 and b0 <= b1 <= tokens else 0
    return b0, n, int(used[z]) - n


def way(parent, b0, i):
    """Node i and those above it, from itself to its root."""
    nodes = [i]
    while 0 <= parent[b0 + nodes[-1]] < nodes[-1]:
        nodes.append(int(parent[b0 + nodes[-1]]))
    return nodes


def places(cu, used, parent, table, tokens, block_size, pages, positions=None):
    """Per token: (sequence, position, page, row); sequence -1: left out, page
    -1: no cache row."""
    out = [(-1, 0, -1, 0)] * tokens
    for z in range(len(used)):
        b0, n, base = bounds(cu, used, tokens, z)
        for i in range(n):
            pos, slot = base + len(way(parent, b0, i)) - 1, base + i
            if pos < 0 or (positions is not None and pos >= positions):
                continue
            e = slot // block_size
            page = int(table[z, e]) if e < table.shape[1] else -1
            out[b0 + i] = (z, pos, page if 0 <= page < pages else -1, slot % block_size)
    return out


def seen(cu, used, parent, table, tokens, block_size, pages, left, most, z):
    """Per node of sequence z that takes part: its keys as (page, row)."""
    b0, n, base = bounds(cu, np.maximum(used, 0), tokens, z)
    out = []
    for i in range(min(n, most)):
        up = way(parent, b0, i)
        depth = len(up) - 1
        keys = range(0 if left < 0 else max(0, base + depth - left), max(base, 0))
        keys = list(keys) + [base + x for k, x in enumerate(up) if (left < 0 or k <= left) and base + x >= 0]
        at = []
        for j in keys:
            e = j // block_size
            page = int(table[z, e]) if e < table.shape[1] else -1
            if 0 <= page < pages:
                at.append((page, j % block_size))
        out.append(at)
    return out


def attention(q, k_cache, v_cache, cu, used, parent, table, scale, left, most):
    """o, lse [h, tokens], rows written, and what the outputs' bars need: per (token, head) the
    largest sum |q k| of a score, the largest |score| and its keys; per (token, head, dim) sum p |V|
    and sum |V| over the keys."""
    t, h, d = q.shape
    pages, bs, hk = k_cache.shape[:3]
    o, lse, rows = np.zeros((t, h, d)), np.full((h, t), np.inf), np.zeros(t, bool)
    qk, top, keys = np.zeros((t, h)), np.zeros((t, h)), np.zeros((t, h))
    pv, av = np.zeros((t, h, d)), np.zeros((t, h, d))
    q, g = q.astype(np.float64), h // hk
    for z in range(len(used)):
        b0 = int(cu[z])
        for i, at in enumerate(seen(cu, used, parent, table, t, bs, pages, left, most, z)):
            r = b0 + i
            rows[r] = True
            if not at:
                continue
            pg, rw = np.array(at).T
            for c in range(hk):
                k, v = k_cache[pg, rw, c].astype(np.float64), v_cache[pg, rw, c].astype(np.float64)
                hs = slice(c * g, (c + 1) * g)
                s = q[r, hs] @ k.T * scale
                m = s.max(-1, keepdims=True)
                e = np.exp(s - m)
                p = e / e.sum(-1, keepdims=True)
                o[r, hs], lse[hs, r] = p @ v, (m + np.log(e.sum(-1, keepdims=True)))[:, 0]
                qk[r, hs] = (np.abs(q[r, hs]) @ np.abs(k).T).max(-1) * abs(scale)
                top[r, hs], keys[r, hs] = np.abs(s).max(-1), len(at)
                pv[r, hs], av[r, hs] = p @ np.abs(v), np.abs(v).sum(0) / e.sum(-1, keepdims=True)
    return o, lse, rows, dict(qk=qk, top=top, keys=keys, pv=pv, av=av)


def verify(target, draft, tokens, parent, u, last, cu, most, distinct, nodes=1024):
    """path [b, most], count and next token of each sequence, the residual
    distribution kept as it stands and normalised after each refusal."""
    b, v = len(cu) - 1, target.shape[1]
    clean = lambda x: np.maximum(np.nan_to_num(x.astype(np.float64), nan=0.0, posinf=np.inf), 0.0)  # noqa: E731
    path, count, nxt = np.full((b, most), -1, np.int64), np.zeros(b, np.int64), np.full(b, -1, np.int64)
    for z in range(b):
        b0, n, _ = bounds(cu, np.zeros(b), target.shape[0], z)
        if n == 0:
            continue
        way_, kept = [0], None
        while len(way_) < most:
            cur = way_[-1]
            p = r = clean(target[b0 + cur])
            q = None if draft is None else clean(draft[b0 + cur])
            got, any_no = None, False
            for i in [i for i in range(1, min(n, nodes)) if 0 <= parent[b0 + i] < i and parent[b0 + i] == cur]:
                x = int(tokens[b0 + i])
                inside = 0 <= x < v
                rx = r[x] if inside else 0.0
                qx = 1.0 if q is None else q[x] if inside else 0.0
                if float(u[b0 + i]) * qx < rx:
                    got = i
                    break
                any_no = True
                if q is None:
                    r = r.copy()
                    if inside:
                        r[x] = 0.0
                    r = r / (1.0 - rx)
                else:
                    r = np.maximum(r - q, 0.0)
                    r = r / r.sum() if r.sum() > 0 else r
                    if distinct:
                        left = max(1.0 - qx, 2.0 ** -24)
                        q = q.copy()
                        if inside:
                            q[x] = 0.0
                        q = q / left
            if got is None:
                kept = r if any_no and r.sum() > 0 else p
                break
            way_.append(got)
        if kept is None:
            kept = clean(target[b0 + way_[-1]])
        c = np.cumsum(kept)
        path[z, :len(way_)], count[z] = way_, len(way_)
        over = np.flatnonzero(c > float(last[z]) * c[-1])
        some = np.flatnonzero(kept > 0)
        nxt[z] = over[0] if len(over) else some[-1] if len(some) else 0
    return path, count, nxt


def keep(cache, cu, used, table, path, count, tokens=1 << 30):
    """The cache [.., pages, block_size, hk, d] with the paths' rows moved, and
    the keys that are left."""
    out, left = cache.copy(), np.array(used)
    pages, bs = cache.shape[-4:-2]
    for z in range(len(used)):
        _, n, base = bounds(cu, used, tokens, z)
        c = min(max(int(count[z]), 0), path.shape[1], n)
        left[z] = int(used[z]) - n + c

        def at(j):
            e = j // bs
            page = int(table[z, e]) if 0 <= j and e < table.shape[1] else -1
            return (page, j % bs) if 0 <= page < pages else None

        for i in range(c):
            x = int(path[z, i])
            if i <= x < n and at(base + i) and at(base + x):
                (p1, r1), (p0, r0) = at(base + i), at(base + x)
                out[..., p1, r1, :, :] = cache[..., p0, r0, :, :]
    return out, left
