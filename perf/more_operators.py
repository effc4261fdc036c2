"""A decoding step over a tree of drafted tokens: the tree's keys and values
appended to a paged cache, attention of its nodes over the cache, the drafts
verified against the target's probabilities, and the accepted path's cache rows
moved to where they belong.

``listed()`` names twelve cases, ``draw(rng)`` gives further ones of the same
ranges.  ``run`` makes one call: in elementary torch operations, or, where
``own`` is true, through ``compiler_amd.operators``.  ``exact`` is the same
result in 64 bits.

A sequence's n nodes are rows cu[z] .. cu[z + 1] - 1; ``parent`` holds each
node's parent as an index within the sequence, below its own, or -1.  With base =
used - n keys before them, node i's key lies in cache row base + i and stands at position
base + depth(i).
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # the drafts of a small batch, small heads, adjacent pairs
        {"name": "append_small", "op": "append", "b": 3, "h": 16, "hk": 4, "d": 64, "dtype": "f16", "n_max": 17,
         "n_min": 5, "k_max": 2051, "k_min": 77, "page": 16, "interleaved": True},
        # wide trees of a large batch
        {"name": "append_wide", "op": "append", "b": 64, "h": 32, "hk": 8, "d": 128, "dtype": "bf16", "n_max": 64,
         "n_min": 40, "k_max": 1024, "k_min": 130, "page": 64, "interleaved": False},
        # the single-token form: no drafts, one node a sequence
        {"name": "attend_token", "op": "attend", "b": 32, "h": 32, "hk": 8, "d": 128, "dtype": "bf16", "n_max": 1,
         "n_min": 1, "k_max": 4096, "k_min": 300, "page": 64, "left": -1},
        # one user, one tree: latency
        {"name": "attend_one", "op": "attend", "b": 1, "h": 32, "hk": 8, "d": 128, "dtype": "bf16", "n_max": 26,
         "n_min": 26, "k_max": 1000, "k_min": 1000, "page": 64, "left": -1},
        # a batch of trees at different positions
        {"name": "attend_step", "op": "attend", "b": 16, "h": 32, "hk": 8, "d": 128, "dtype": "bf16", "n_max": 32,
         "n_min": 9, "k_max": 4096, "k_min": 300, "page": 64, "left": -1},
        # wide trees over long contexts: as many products as bytes
        {"name": "attend_wide", "op": "attend", "b": 8, "h": 32, "hk": 8, "d": 128, "dtype": "bf16", "n_max": 64,
         "n_min": 50, "k_max": 8192, "k_min": 2049, "page": 64, "left": -1},
        # long documents, eight small heads on one KV head, small pages
        {"name": "attend_long", "op": "attend", "b": 2, "h": 8, "hk": 1, "d": 64, "dtype": "f16", "n_max": 13,
         "n_min": 7, "k_max": 65537, "k_min": 50001, "page": 16, "left": -1},
        # one user's tree, each level drawn from the draft's row with replacement
        {"name": "verify_one", "op": "verify", "b": 1, "v": 32000, "dtype": "f32", "n_max": 26, "n_min": 26,
         "drafts": "drawn"},
        # a batch over a large vocabulary, siblings drawn without replacement
        {"name": "verify_step", "op": "verify", "b": 16, "v": 128000, "dtype": "f32", "n_max": 26, "n_min": 9,
         "drafts": "distinct"},
        # drafts looked up instead of drawn (no draft probabilities), an odd vocabulary in 16 bits
        {"name": "verify_chosen", "op": "verify", "b": 32, "v": 50257, "dtype": "bf16", "n_max": 12, "n_min": 4,
         "drafts": "chosen"},
        # the accepted rows of one layer
        {"name": "keep_layer", "op": "keep", "b": 16, "layers": 1, "hk": 8, "d": 128, "dtype": "bf16", "n_max": 32,
         "n_min": 9, "k_max": 1024, "k_min": 100, "page": 64},
        # of all layers at once
        {"name": "keep_layers", "op": "keep", "b": 32, "layers": 16, "hk": 8, "d": 128, "dtype": "bf16", "n_max": 64,
         "n_min": 26, "k_max": 256, "k_min": 100, "page": 64},
    ]


# ------------------------------------------------------------------ drawing
def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "verify", "verify", "verify", "keep"])
    half = rng.choice(["bf16", "bf16", "f16"])
    n = rng.choice([1, 1 + rng.randrange(8), 8 + rng.randrange(25), 26, 60, 64])
    n_min = max(1, int(n * rng.uniform(0.2, 1.0)))
    if op == "verify":
        v = _log(rng, 1000, 128000)
        if rng.random() < 0.5:
            v = max(8, v // 8 * 8)
        b, n = _log(rng, 1, 32), min(n, 32)
        b = max(1, min(b, 16 * 26 * 128000 // (v * n)))
        return {"op": op, "b": b, "v": v, "dtype": rng.choice(["f32", "f32", half]), "n_max": n, "n_min": min(n, n_min),
                "drafts": rng.choice(["drawn", "distinct", "chosen"])}
    h, hk = rng.choice([(32, 8), (32, 8), (32, 4), (16, 4), (8, 8), (8, 1)])
    case = {"op": op, "b": 1, "h": h, "hk": hk, "d": rng.choice([128, 128, 64]), "dtype": half, "n_max": n, "n_min": n_min}
    page = rng.choice([16, 32, 64, 64, 128])
    if op == "keep":
        case.pop("h")
        b, layers, k = _log(rng, 1, 32), _log(rng, 1, 16), n + _log(rng, 1, 190)
        return dict(case, b=b, layers=layers, k_max=k, k_min=max(n, int(k * rng.uniform(0.3, 1.0))), page=page)
    if op == "append":
        b, k = _log(rng, 1, 64), n + _log(rng, 1, 960)
        return dict(case, b=b, k_max=k, k_min=max(n, int(k * rng.uniform(0.05, 1.0))), page=page,
                    interleaved=rng.random() < 0.3)
    b = _log(rng, 1, 32)
    k = n + _log(rng, 8, min(65000, 8 * 56 * 5000 * 32 // (b * max(n, 8) * h), 32 * 2100 * 8 // (b * hk)))
    return dict(case, b=b, k_max=k, k_min=max(n, int(k * rng.uniform(0.05, 1.0))), page=page,
                left=rng.choice([-1, -1, -1, 1000]))


# ------------------------------------------------------------------- inputs
def _lengths(case, hi, lo):
    b = case["b"]
    return [case[hi] if b == 1 else case[hi] - (case[hi] - case[lo]) * i // (b - 1) for i in range(b)]


def _trees(case, seed):
    """Each sequence's parents: breadth first, levels of a few children a node."""
    r, trees = random.Random(seed), []
    for n in _lengths(case, "n_max", "n_min"):
        p = [-1]
        for i in range(1, n):
            p.append(0 if i < 3 else min(i - 1, p[-1] + r.choice([0, 0, 0, 1, 1])))
        trees.append(p)
    return trees


def _walk(p, i):
    """Nodes from the root to node i."""
    path = []
    while i >= 0:
        path.append(i)
        i = p[i]
    return path[::-1]


def _kept(trees, seed):
    """An accepted path of each tree.  (Of those whose rows the move does not overwrite, so that
    a pass can be made again on the same cache.)"""
    r, paths = random.Random(seed + 1), []
    for p in trees:
        all_ = [_walk(p, i) for i in range(len(p))]
        fit = [w for w in all_ if all(x == i or x >= len(w) for i, x in enumerate(w))]
        long = [w for w in fit if len(w) >= min(3, max(map(len, fit)))]
        paths.append(r.choice(long))
    return paths


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    ints = lambda v, t=torch.int32: torch.tensor(v, dtype=t).to("cuda")  # noqa: E731

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=g, device="cuda") * std

    trees = _trees(case, seed)
    nl = [len(p) for p in trees]
    tokens = sum(nl)
    state = {"case": dict(case), "cu": ints([sum(nl[:i]) for i in range(len(nl) + 1)]),
             "parent": ints([x for p in trees for x in p]), "nodes": max(nl)}
    if case["op"] == "verify":
        v = case["v"]
        x = normal(tokens, v, std=3.0)
        draft = torch.softmax(0.9 * x + normal(tokens, v), -1).to(dt)
        state["target"] = torch.softmax(x, -1).to(dt)
        x = None
        # each node's token from its parent's row; siblings of equal rank at once
        first = [0] * tokens
        rank, at = [0] * tokens, 0
        for p in trees:
            for i in range(1, len(p)):
                first[at + i] = at + p[i]
                rank[at + i] = sum(q == p[i] for q in p[1:i])
            at += len(p)
        if case["drafts"] == "chosen":  # looked up: often what the target holds likely
            state["token"] = torch.zeros(tokens, dtype=torch.int64, device="cuda")
            top = torch.topk(state["target"].float(), 4).indices
        else:
            state["token"] = torch.randint(0, v, (tokens,), generator=g, device="cuda")
        for k in range(max(rank) + 1):
            rows = [t for t in range(tokens) if rank[t] == k]
            src, rows = ints([first[t] for t in rows], torch.int64), ints(rows, torch.int64)
            if case["drafts"] == "chosen":
                state["token"][rows] = top[src, min(k, 3)] if k else top[src, 0]
                continue
            w = draft[src].float()
            if case["drafts"] == "distinct":
                w = w + 1e-30
                for j in range(k):  # earlier siblings' tokens are gone
                    gone = ints([t for s in rows.tolist() for t in [next(
                        u for u in range(s) if first[u] == first[s] and rank[u] == j and u != first[u])]], torch.int64)
                    w.scatter_(1, state["token"][gone][:, None], 0.0)
            state["token"][rows] = torch.multinomial(w, 1, generator=g)[:, 0]
        state["draft"] = None if case["drafts"] == "chosen" else draft
        state["u"] = torch.rand(tokens, generator=g, device="cuda")
        state["last"] = torch.rand(case["b"], generator=g, device="cuda")
        state["depth"], state["children"] = min(case["n_max"], 16), max(1, *(p.count(i) for p in trees for i in range(len(p))))
        return state
    kl = _lengths(case, "k_max", "k_min")
    kl = [max(k, n) for k, n in zip(kl, nl)]
    hk, d, page = case["hk"], case["d"], case["page"]
    # pages of the sequences in shuffled order
    per = [(n + page - 1) // page for n in kl]
    pages = sum(per)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    start = ints([sum(per[:i]) for i in range(len(per))])
    col = torch.arange(max(per), device="cuda")[None, :]
    table = torch.where(col < ints(per)[:, None], order[(start[:, None] + col).clamp(max=pages - 1)], -1)
    state.update(used=ints(kl), table=table.to(torch.int32).contiguous(), seqlen_k=max(kl))
    if case["op"] == "keep":
        paths = _kept(trees, seed)
        wide = max(len(w) for w in paths) + 1
        state["path"] = ints([w + [-1] * (wide - len(w)) for w in paths])
        state["count"] = ints([len(w) for w in paths])
        shape = (case["layers"], pages, page, hk, d)[0 if case["layers"] > 1 else 1:]
        state["k_cache"], state["v_cache"] = normal(*shape).to(dt), normal(*shape).to(dt)
        return state
    h = case["h"]
    if case["op"] == "attend":
        # keys have a few channels far larger than the others
        big = torch.where(torch.rand(d, generator=g, device="cuda") < 0.05, 4.0, 1.0)
        state["k_cache"] = normal(pages, page, hk, d).mul_(big).to(dt)
        state["v_cache"] = normal(pages, page, hk, d).to(dt)
        state["q"] = normal(tokens, h, d).to(dt)
        return state
    # one projection's output holds a token's queries, keys and values
    qkv = normal(tokens, (h + 2 * hk) * d).to(dt).view(tokens, h + 2 * hk, d)
    state["q"], state["k"], state["v"] = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
    angle = torch.arange(max(kl), device="cuda").double()[:, None] * 10000.0 ** (
        -torch.arange(0, d, 2, device="cuda").double() / d)
    state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    state["k_cache"] = torch.zeros((pages, page, hk, d), dtype=dt, device="cuda")
    state["v_cache"] = torch.zeros_like(state["k_cache"])
    return state


# ---------------------------------------------------------------- plain form
def _places(s, tokens):
    """Sequence, index and base of each node."""
    t = torch.arange(tokens, device="cuda")
    seq = (t[:, None] >= s["cu"][None, 1:]).sum(-1)
    return seq, t - s["cu"][seq], s["used"][seq].long() - s["cu"][seq + 1] + s["cu"][seq]


def _above(s, seq, i):
    """[tokens, nodes]: whether a node of the same sequence is the token's own or above it."""
    n, b = s["nodes"], s["used"].shape[0]
    up = torch.eye(n, device="cuda").repeat(b, 1, 1)
    has = s["parent"] >= 0
    up[seq[has], i[has].long(), s["parent"][has].long()] = 1.0
    for _ in range((n - 1).bit_length()):  # paths of twice the length
        up = torch.matmul(up, up).clamp(max=1.0)
    return up[seq, i.long()] > 0


def _append(s):
    case, dt, page = s["case"], s["q"].dtype, s["case"]["page"]
    seq, i, base = _places(s, s["q"].shape[0])
    pos = base + _above(s, seq, i).sum(-1) - 1
    at, row = s["table"][seq, (base + i) // page].long(), (base + i) % page
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]

    def turn(x):
        x, half = x.float(), x.shape[-1] // 2
        a, b = (x[..., 0::2], x[..., 1::2]) if case["interleaved"] else (x[..., :half], x[..., half:])
        y, z = a * cos - b * sin, b * cos + a * sin
        return (torch.stack([y, z], -1).flatten(-2) if case["interleaved"] else torch.cat([y, z], -1)).to(dt)

    s["k_cache"][at, row], s["v_cache"][at, row] = turn(s["k"]), s["v"]
    return {"q": turn(s["q"]), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _attend(s):
    case = s["case"]
    b, h, hk, d, page, left = (case[n] for n in ("b", "h", "hk", "d", "page", "left"))
    nq, nk, g = s["nodes"], s["seqlen_k"], h // hk
    tokens = s["q"].shape[0]
    seq, i, base = _places(s, tokens)
    up = _above(s, seq, i)
    j = torch.arange(nk, device="cuda")
    at = s["table"][:, j // page].clamp(min=0).long()  # [b, keys]
    kt = s["k_cache"][at, j % page].float().permute(0, 2, 3, 1).contiguous()  # [b, hk, d, keys]
    v = s["v_cache"][at, j % page].float().permute(0, 2, 1, 3).contiguous()
    rows = (s["cu"][:-1, None] + torch.arange(nq, device="cuda")).clamp(max=tokens - 1).long()
    q = s["q"][rows].float().view(b, nq, hk, g, d).permute(0, 2, 3, 1, 4).reshape(b, hk, g * nq, d)
    p = torch.matmul(q, kt).mul_(1.0 / math.sqrt(d)).view(b, hk, g, nq, nk)
    # a key before the tree, or the node's own or one above it
    depth = up.sum(-1) - 1
    node = (j - base[:, None])  # [tokens, keys]
    see = torch.where(node < 0, True, up.gather(1, node.clamp(0, nq - 1)) & (node < nq))
    if left >= 0:
        height = torch.zeros_like(up, dtype=torch.int64).copy_(up).cumsum(-1) - 1  # depth of those above
        pos = torch.where(node < 0, j.expand_as(node), base[:, None] + height.gather(1, node.clamp(0, nq - 1)))
        see &= pos >= (base + depth - left)[:, None]
    p.masked_fill_(~see[rows][:, None, None], -math.inf)
    m = p.amax(-1, keepdim=True).clamp(min=-3e38)
    p.sub_(m).exp_()
    z = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(b, hk, g * nq, nk), v).view(b, hk, g, nq, d) / z
    lse = (m + z.log()).squeeze(-1)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, nq, h, d)[seq, i].to(s["q"].dtype)
    return {"o": o, "lse": lse.reshape(b, h, nq).permute(0, 2, 1)[seq, i].t()}


def _verify(s):
    """All nodes' children of equal rank at once, then the way from each root."""
    b, tokens, given = s["case"]["b"], s["token"].shape[0], s["draft"] is not None
    t = torch.arange(tokens, device="cuda")
    start = s["cu"][:-1].long()
    of = (t[:, None] >= s["cu"][None, 1:]).sum(-1)
    above = torch.where(s["parent"] >= 0, start[of] + s["parent"], tokens)  # row of the parent
    rank = ((above[:, None] == above[None, :]) & (t[None, :] < t[:, None])).sum(-1)
    child = torch.full((tokens + 1, s["children"]), -1, dtype=torch.int64, device="cuda")
    child[above, torch.where(s["parent"] >= 0, rank, 0)] = t
    child = child[:tokens]
    p = s["target"].double()
    q = s["draft"].double() if given else None
    taken = torch.zeros(tokens, dtype=torch.float64, device="cuda")
    total, rest, to = taken + 1, taken + 1, torch.full_like(t, -1)
    for k in range(s["children"]):
        mine = (child[:, k] >= 0) & (to < 0)
        c = child[:, k].clamp(min=0)
        x = s["token"][c]
        qx = q[t, x] if given else taken + 1
        left = (p[t, x] - taken * qx).clamp(min=0) if given else p[t, x]
        yes = mine & (s["u"][c].double() * qx * total < left * rest)
        no = mine & ~yes
        to = torch.where(yes, c, to)
        # refused: what the target has more than the draft took away
        if not given:
            total = torch.where(no, total - left, total)
            p[t, x] = torch.where(no, 0.0, left)
            continue
        taken = torch.where(no, taken + total / rest, taken)
        total = torch.where(no, torch.addcmul(p, taken[:, None], q, value=-1).clamp_(min=0).sum(-1), total)
        if s["case"]["drafts"] == "distinct":
            rest = torch.where(no, (rest - qx).clamp(min=2.0 ** -24), rest)
    at, count = start, torch.ones_like(start)
    path = torch.full((b, s["depth"]), -1, dtype=torch.int32, device="cuda")
    path[:, 0] = 0
    for k in range(1, s["depth"]):
        on = (to[at] >= 0) & (count == k)
        at, count = torch.where(on, to[at], at), count + on
        path[:, k] = torch.where(on, at - start, -1)
    # at the path's full length the last node's children are not looked at
    full = count == s["depth"]
    left = p[at] if not given else torch.where((taken[at] * ~full)[:, None] > 0, p[at] - taken[at][:, None] * q[at], p[at])
    left = torch.where(full[:, None], s["target"][at].double(), left.clamp(min=0))
    left = torch.where(left.sum(-1, keepdim=True) > 0, left, s["target"][at].double())  # nothing left
    sums = left.cumsum(-1)
    token = (sums <= s["last"].double()[:, None] * sums[:, -1:]).sum(-1)
    return {"path": path, "count": count.to(torch.int32), "next": token}


def _keep(s):
    page = s["case"]["page"]
    base = (s["used"] - s["cu"][1:] + s["cu"][:-1]).long()[:, None]
    i = torch.arange(s["path"].shape[1], device="cuda")[None, :]
    move = i < s["count"][:, None]
    src, dst = base + torch.where(move, s["path"], 0), base + torch.where(move, i, 0)
    seq = torch.arange(base.shape[0], device="cuda")[:, None]
    a, c = s["table"][seq, src // page].long(), s["table"][seq, dst // page].long()
    for cache in (s["k_cache"], s["v_cache"]):
        layers = cache if cache.dim() == 5 else cache[None]
        layers[:, c, dst % page] = layers[:, a, src % page]
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "used": base[:, 0].to(torch.int32) + s["count"]}


# ---------------------------------------------------------------- one pass
def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        return {"append": _append, "attend": _attend, "verify": _verify, "keep": _keep}[op](s)
    from compiler_amd import operators as ops
    if op == "append":
        q = ops.paged_append_tree(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["k_cache"], s["v_cache"], s["table"],
                                  s["cu"], s["used"], s["parent"], interleaved=case["interleaved"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if op == "attend":
        o, lse = ops.paged_attention_tree(s["q"], s["k_cache"], s["v_cache"], s["table"], s["cu"], s["used"], s["parent"],
                                          s["nodes"], s["seqlen_k"], window_left=case["left"])
        return {"o": o, "lse": lse}
    if op == "verify":
        path, count, token = ops.verify_tree(s["target"], s["draft"], s["token"], s["parent"], s["u"], s["last"], s["cu"],
                                             s["depth"], distinct=case["drafts"] == "distinct")
        return {"path": path, "count": count, "next": token}
    used = ops.paged_keep_path(s["k_cache"], s["v_cache"], s["table"], s["cu"], s["used"], s["path"], s["count"])
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "used": used}


# --------------------------------------------------------------------- work
def work(case):
    e, op = SIZE[case["dtype"]], case["op"]
    nl = _lengths(case, "n_max", "n_min")
    t, b = sum(nl), case["b"]
    if op == "verify":  # the last node's row of the target and, where drawn, of the draft
        rows = 1 if case["drafts"] == "chosen" else 2
        return {"bytes": b * rows * case["v"] * e + 20 * t + 8 * b, "flops": b * rows * case["v"] * 2}
    kl = [max(k, n) for k, n in zip(_lengths(case, "k_max", "k_min"), nl)]
    hk, d, page = case["hk"], case["d"], case["page"]
    if op == "keep":  # two rows of each path move (its root stays)
        return {"bytes": 4 * 2 * sum(min(2, n - 1) for n in nl) * case["layers"] * hk * d * e + 4 * 8 * b, "flops": 0}
    h = case["h"]
    lists = 4 * (2 * b + 1 + t)
    if op == "append":
        lists += 4 * sum((k - 1) // page - (k - n) // page + 1 for n, k in zip(nl, kl))
        # about four levels of each tree take a row of the tables
        return {"bytes": 2 * t * (h + 2 * hk) * d * e + 4 * d * sum(min(4, n) for n in nl) + lists,
                "flops": 3 * t * (h + hk) * d}
    # a node sees the keys before the tree and a few nodes
    seen = lambda k, n: min(k - n, case["left"]) if case["left"] >= 0 else k - n  # noqa: E731
    pairs = sum(n * (seen(k, n) + min(4, n)) for n, k in zip(nl, kl))
    keys = sum(seen(k, n) + n for n, k in zip(nl, kl))
    return {"bytes": 2 * t * h * d * e + 4 * h * t + 2 * keys * hk * d * e + lists + 4 * sum(-(-k // page) for k in kl),
            "flops": 4 * h * d * pairs}


# -------------------------------------------------------------------- exact
def exact(case, seed):
    s, trees = prepare(case, seed), _trees(case, seed)
    op, at = case["op"], 0
    if op == "verify":
        return _exact_verify(case, s, trees)
    kl = s["used"].tolist()
    hk, d, page = case["hk"], case["d"], case["page"]
    if op == "keep":
        out = {n: s[n].double() for n in ("k_cache", "v_cache")}
        for z, w in enumerate(_kept(trees, seed)):
            base, row = kl[z] - len(trees[z]), s["table"][z].tolist()
            for i, x in enumerate(w):
                for n, c in out.items():
                    c[..., row[(base + i) // page], (base + i) % page, :, :] = s[n][
                        ..., row[(base + x) // page], (base + x) % page, :, :].double()
        return dict(out, used=torch.tensor([k - len(p) + len(w) for k, p, w in zip(kl, trees, _kept(trees, seed))],
                                           dtype=torch.int32, device="cuda"))
    depth = [[len(_walk(p, i)) - 1 for i in range(len(p))] for p in trees]
    if op == "append":
        pos = torch.tensor([k - len(p) + x for k, p, ds in zip(kl, trees, depth) for x in ds], device="cuda")
        seq = torch.tensor([z for z, p in enumerate(trees) for _ in p], device="cuda")
        slot = torch.tensor([k - len(p) + i for k, p in zip(kl, trees) for i in range(len(p))], device="cuda")
        # the tables are inputs: their angle, with the size that their rounding gives them left in
        c, n = s["cos"][pos].double(), s["sin"][pos].double()
        unit = torch.complex(c, n)[:, None]

        def turn(x):
            x, half = x.double(), d // 2
            pair = x.unflatten(-1, (half, 2)) if case["interleaved"] else x.unflatten(-1, (2, half)).transpose(-1, -2)
            y = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * unit)
            return y.flatten(-2) if case["interleaved"] else y.transpose(-1, -2).flatten(-2)

        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        place = (s["table"][seq, slot // page].long(), slot % page)
        kc[place], vc[place] = turn(s["k"]), s["v"].double()
        return {"q": turn(s["q"]), "k_cache": kc, "v_cache": vc}
    h, g, left = case["h"], case["h"] // hk, case["left"]
    o = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty((h, s["q"].shape[0]), dtype=torch.float64, device="cuda")
    for z, p in enumerate(trees):
        n, nk = len(p), kl[z]
        base = nk - n
        hide = torch.zeros(n, nk, dtype=torch.bool)
        hide[:, base:] = True
        for i in range(n):
            hide[i, [base + x for x in _walk(p, i)]] = False
            if left >= 0:
                hide[i, :max(0, min(base, base + depth[z][i] - left))] = True
                hide[i, [base + x for x in _walk(p, i) if depth[z][x] < depth[z][i] - left]] = True
        hide = hide.to("cuda")
        used = s["table"][z, :(nk + page - 1) // page].long()
        for c in range(hk):
            k, v = (x[used, :, c].double().reshape(-1, d)[:nk] for x in (s["k_cache"], s["v_cache"]))
            heads = slice(c * g, (c + 1) * g)
            w = torch.matmul(s["q"][at:at + n, heads].double().transpose(0, 1).reshape(-1, d), k.t()) / math.sqrt(d)
            w = w.view(g, n, nk).masked_fill(hide, -math.inf)
            lse[heads, at:at + n] = torch.logsumexp(w, -1)
            o[at:at + n, heads] = (torch.softmax(w, -1).reshape(-1, nk) @ v).view(g, n, d).transpose(0, 1)
        at += n
    return {"o": o, "lse": lse}


def _exact_verify(case, s, trees):
    """Sequence by sequence: the residual distribution as it stands, normalised after each refusal."""
    token, u, last = s["token"].tolist(), s["u"].double().tolist(), s["last"].double().tolist()
    path = torch.full((case["b"], s["depth"]), -1, dtype=torch.int32)
    count, nxt, at = [], [], 0
    for z, p in enumerate(trees):
        way = [0]
        while True:
            target = s["target"][at + way[-1]].double()
            r, draft = target, None if s["draft"] is None else s["draft"][at + way[-1]].double()
            plain = True  # the rows count as normalised until something is refused
            got = None
            for i in [i for i in range(1, len(p)) if p[i] == way[-1]]:
                x = token[at + i]
                dx = 1.0 if draft is None else float(draft[x])
                if u[at + i] * dx < float(r[x]):
                    got = i
                    break
                if draft is None:
                    scale = 1.0 - float(r[x])
                    r = r.clone()
                    r[x] = 0.0
                    r = r / scale
                else:
                    r = torch.relu(r - draft)
                    r = r / r.sum()
                    if case["drafts"] == "distinct":
                        draft = draft.clone()
                        left = max(1.0 - dx, 2.0 ** -24)
                        draft[x] = 0.0
                        draft = draft / left
                plain = False
            if got is None:
                break
            way.append(got)
            if len(way) == s["depth"]:  # no room for more: the last node's children are not looked at
                target, plain = s["target"][at + way[-1]].double(), True
                r = target
                break
        if not plain and not float(r.nan_to_num().sum()) > 0:
            r = target
        sums = r.cumsum(0)
        nxt.append(int((sums <= last[z] * sums[-1]).sum()))
        count.append(len(way))
        path[z, :len(way)] = torch.tensor(way, dtype=torch.int32)
        at += len(p)
    return {"path": path.to("cuda"), "count": torch.tensor(count, dtype=torch.int32, device="cuda"),
            "next": torch.tensor(nxt, device="cuda")}
