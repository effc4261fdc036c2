"""A layer's step over a paged cache: appending keys and values (16 and 4 bits)
with the position rotation, attention over the 4-bit cache, and the norms
around a block with its gate and residual.

``listed()`` names twelve cases, ``draw(rng)`` gives further ones of the same
ranges.  ``run`` makes one call: in elementary torch operations, or, where
``own`` is true, through ``compiler_amd.operators``.  ``exact`` is the same
result in 64 bits.

The 4-bit cache holds a (token, head) row as codes c of 4 bits (dim 2i in the
low half of byte i, dim 2i + 1 in the high half) and a pair (s, o) of the
model's type: the row's values are (c - 8) s + o, with s = (max - min) / 15 and
o = min + 8 s, each rounded to the model's type.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-6


def listed():
    return [
        # one decoding step of a batch at different positions, 16-bit cache
        {"name": "append_step", "op": "append", "b": 32, "h": 32, "hk": 8, "d": 128, "dtype": "bf16", "q_max": 1,
         "q_min": 1, "k_max": 4096, "k_min": 300, "page": 64, "interleaved": False},
        # whole prompts of different lengths, packed
        {"name": "append_prompt", "op": "append", "b": 8, "h": 32, "hk": 8, "d": 128, "dtype": "bf16",
         "q_max": 4096, "q_min": 2304, "k_max": 4096, "k_min": 2304, "page": 64, "interleaved": False},
        # one to five tokens a sequence (drafts to verify) into 4 bits, small heads, adjacent pairs
        {"name": "append_int4_draft", "op": "append4", "b": 13, "h": 16, "hk": 4, "d": 64, "dtype": "f16",
         "q_max": 5, "q_min": 1, "k_max": 2051, "k_min": 77, "page": 16, "interleaved": True},
        # prompts into the 4-bit cache
        {"name": "append_int4_prompt", "op": "append4", "b": 8, "h": 32, "hk": 8, "d": 128, "dtype": "bf16",
         "q_max": 2048, "q_min": 333, "k_max": 2048, "k_min": 333, "page": 64, "interleaved": False},
        # one user, one token: latency
        {"name": "attend_one", "op": "attend4", "b": 1, "h": 32, "hk": 8, "d": 128, "dtype": "bf16", "q_max": 1,
         "q_min": 1, "k_max": 1000, "k_min": 1000, "page": 64, "causal": True},
        # a decoding step of a batch at different positions
        {"name": "attend_step", "op": "attend4", "b": 32, "h": 32, "hk": 8, "d": 128, "dtype": "bf16", "q_max": 1,
         "q_min": 1, "k_max": 4096, "k_min": 300, "page": 64, "causal": True},
        # verifying four drafted tokens, eight heads on one KV head, small pages
        {"name": "attend_draft", "op": "attend4", "b": 16, "h": 8, "hk": 1, "d": 64, "dtype": "f16", "q_max": 4,
         "q_min": 4, "k_max": 8192, "k_min": 511, "page": 16, "causal": True},
        # long documents: few sequences, many keys
        {"name": "attend_long", "op": "attend4", "b": 3, "h": 32, "hk": 8, "d": 128, "dtype": "bf16", "q_max": 1,
         "q_min": 1, "k_max": 81920, "k_min": 65537, "page": 64, "causal": True},
        # a chunk of a prompt behind a cached prefix
        {"name": "attend_chunk", "op": "attend4", "b": 2, "h": 32, "hk": 8, "d": 128, "dtype": "bf16", "q_max": 512,
         "q_min": 301, "k_max": 4096, "k_min": 3001, "page": 64, "causal": True},
        # between two blocks of a decoding step
        {"name": "norm_step", "op": "norm", "rows": 16, "cols": 4096, "dtype": "bf16", "post": True, "gate": "none",
         "act": "none", "alpha": 1.0},
        # the same over a long prompt, a learned gate per channel, rows that are no power of two
        {"name": "norm_prompt", "op": "norm", "rows": 8191, "cols": 3000, "dtype": "bf16", "post": True,
         "gate": "channel", "act": "none", "alpha": 1.0},
        # a computed gate for every value, in fp32, with a scaled residual
        {"name": "norm_gated", "op": "norm", "rows": 4096, "cols": 4096, "dtype": "f32", "post": True, "gate": "full",
         "act": "sigmoid", "alpha": 0.5},
    ]


# ------------------------------------------------------------------ drawing
def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "append4", "append4", "attend4", "attend4", "attend4", "norm", "norm"])
    half = rng.choice(["bf16", "bf16", "f16"])
    if op == "norm":
        rows, cols = _log(rng, 1, 8192), _log(rng, 256, 8192)
        if rng.random() < 0.7:
            cols = max(8, cols // 8 * 8)
        dtype = rng.choice([half, half, half, "f32"])
        if rows * cols * SIZE[dtype] > 4096 * 4096 * 4:
            rows = 4096 * 4096 * 4 // (cols * SIZE[dtype])
        gate = rng.choice(["none", "channel", "row", "full"])
        return {"op": op, "rows": rows, "cols": cols, "dtype": dtype, "post": rng.random() < 0.8, "gate": gate,
                "act": rng.choice(["none", "sigmoid", "tanh"]) if gate != "none" else "none",
                "alpha": rng.choice([1.0, 1.0, 0.5, 1.25])}
    h, hk = rng.choice([(32, 8), (32, 32), (16, 4), (8, 8), (8, 1)])
    d = rng.choice([128, 128, 64])
    page = rng.choice([16, 32, 64, 64, 128])
    case = {"op": op, "b": 1, "h": h, "hk": hk, "d": d, "dtype": half}
    many = rng.random() < 0.4
    if op == "attend4":
        if many:  # chunks of prompts
            b, q = _log(rng, 1, 4), _log(rng, 8, 512)
            k = _log(rng, q, max(q, min(8192, 2 * 32 * 512 * 4096 // (b * h * q))))
        else:
            b, q = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 4, 5])
            k = _log(rng, 8, min(65536, 3 * 65536 * 8 // (b * hk)))
        q = min(q, k)
        return dict(case, b=b, q_max=q, q_min=max(1, int(q * rng.uniform(0.3, 1.0))), k_max=k,
                    k_min=max(q, int(k * rng.uniform(0.05, 1.0))), page=page, causal=rng.random() < 0.8)
    if many:
        b, q = _log(rng, 1, 8), _log(rng, 16, 2048)
        k = q + rng.choice([0, 0, 1, 500])
    else:
        b, q = _log(rng, 1, 64), rng.choice([1, 1, 2, 5])
        k = _log(rng, q, 4096)
    return dict(case, b=b, q_max=q, q_min=max(1, int(q * rng.uniform(0.3, 1.0))), k_max=k,
                k_min=max(q, int(k * rng.uniform(0.05, 1.0))), page=page, interleaved=rng.random() < 0.3)


# ------------------------------------------------------------------- inputs
def _lengths(case):
    """New tokens and cached keys (the new ones among them) of each sequence."""
    b = case["b"]
    step = lambda hi, lo, i: hi if b == 1 else hi - (hi - lo) * i // (b - 1)  # noqa: E731
    return ([step(case["q_max"], case["q_min"], i) for i in range(b)],
            [step(case["k_max"], case["k_min"], i) for i in range(b)])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=g, device="cuda") * std

    if case["op"] == "norm":
        r, c = case["rows"], case["cols"]
        state = {"case": dict(case), "x": normal(r, c, std=2.0).to(dt), "h": normal(r, c, std=0.5).to(dt),
                 "w_pre": (1.0 + normal(c, std=0.2)).to(dt), "w_post": None, "gate": None}
        if case["post"]:
            state["w_post"] = (1.0 + normal(c, std=0.2)).to(dt)
        shape = {"none": None, "channel": (1, c), "row": (r, 1), "full": (r, c)}[case["gate"]]
        if shape:
            state["gate"] = normal(*shape).to(dt)
        return state
    h, hk, d, page = case["h"], case["hk"], case["d"], case["page"]
    ql, kl = _lengths(case)
    ints = lambda v: torch.tensor(v, dtype=torch.int32).to("cuda")  # noqa: E731
    # pages of the sequences in shuffled order
    per = [(n + page - 1) // page for n in kl]
    pages = sum(per)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    first = ints([sum(per[:i]) for i in range(len(per))])
    col = torch.arange(max(per), device="cuda")[None, :]
    table = torch.where(col < ints(per)[:, None], order[(first[:, None] + col).clamp(max=pages - 1)], -1)
    state = {"case": dict(case), "cu": ints([sum(ql[:i]) for i in range(len(ql) + 1)]), "used": ints(kl),
             "table": table.to(torch.int32).contiguous(), "seqlen_q": max(ql), "seqlen_k": max(kl)}
    tokens = sum(ql)
    if case["op"] == "attend4":
        # keys have a few channels far larger than the others
        big = torch.where(torch.rand(d, generator=g, device="cuda") < 0.05, 4.0, 1.0)
        k = normal(pages, hk, page, d).mul_(big)
        state["k_cache"], state["k_scale"] = (x.transpose(1, 2) for x in _pack(*_codes(k, dt), dt))
        k = None
        v = normal(pages, hk, page, d)
        state["v_cache"], state["v_scale"] = (x.transpose(1, 2) for x in _pack(*_codes(v, dt), dt))
        state["q"] = normal(tokens, h, d).to(dt)
        return state
    # one projection's output holds a token's queries, keys and values
    qkv = normal(tokens, (h + 2 * hk) * d).to(dt).view(tokens, h + 2 * hk, d)
    state["q"], state["k"], state["v"] = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
    angle = torch.arange(max(kl), device="cuda").double()[:, None] * 10000.0 ** (
        -torch.arange(0, d, 2, device="cuda").double() / d)
    state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    if case["op"] == "append":
        state["k_cache"] = torch.zeros((pages, page, hk, d), dtype=dt, device="cuda")
        state["v_cache"] = torch.zeros_like(state["k_cache"])
    else:  # a page holds a head's rows together
        for n in ("k", "v"):
            state[n + "_cache"] = torch.zeros((pages, hk, page, d // 2), dtype=torch.uint8, device="cuda").transpose(1, 2)
            state[n + "_scale"] = torch.zeros((pages, hk, page, 2), dtype=dt, device="cuda").transpose(1, 2)
    return state


# ---------------------------------------------------------------- plain form
def _codes(x, dt):
    """4-bit codes, scale and offset of rows x (fp32)."""
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    s = ((hi - lo) / 15).to(dt).float()
    s = torch.where(s < 2.0 ** -126, 0.0, s)
    o = (lo + 8 * s).to(dt).float()
    inv = torch.where(s > 0, 1 / s, 0.0)
    return ((x - o) * inv).round_().add_(8).clamp_(0, 15).to(torch.uint8), s, o


def _pack(c, s, o, dt):
    return c[..., 0::2] | (c[..., 1::2] << 4), torch.cat([s, o], -1).to(dt)


def _values(codes, scale):
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    return (c - 8) * scale[..., :1].float() + scale[..., 1:].float()


def _rotate(x, cos, sin, interleaved):
    """x [tokens, heads, d], cos / sin [tokens, 1, d / 2]."""
    x = x.float()
    d = x.shape[-1]
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :d // 2], x[..., d // 2:])
    y, z = a * cos - b * sin, b * cos + a * sin
    return torch.stack([y, z], -1).flatten(-2) if interleaved else torch.cat([y, z], -1)


def _places(s, tokens):
    """Sequence and position of each token."""
    t = torch.arange(tokens, device="cuda")
    seq = (t[:, None] >= s["cu"][None, 1:]).sum(-1)
    return t, seq, s["used"][seq].long() - s["cu"][seq + 1] + t


def _append(s):
    case, dt, page = s["case"], s["q"].dtype, s["case"]["page"]
    _, seq, pos = _places(s, s["q"].shape[0])
    at, row = s["table"][seq, pos // page].long(), pos % page
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    q = _rotate(s["q"], cos, sin, case["interleaved"]).to(dt)
    k, v = _rotate(s["k"], cos, sin, case["interleaved"]), s["v"].float()
    if case["op"] == "append":
        s["k_cache"][at, row], s["v_cache"][at, row] = k.to(dt), v.to(dt)
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    kp, ks = _pack(*_codes(k, dt), dt)
    vp, vs = _pack(*_codes(v, dt), dt)
    s["k_cache"][at, row], s["k_scale"][at, row] = kp, ks
    s["v_cache"][at, row], s["v_scale"][at, row] = vp, vs
    return {"q": q, "k": _values(kp, ks).to(dt), "v": _values(vp, vs).to(dt), "k_scale": s["k_scale"],
            "v_scale": s["v_scale"]}


def _attend(s):
    case = s["case"]
    b, h, hk, d, page = (case[n] for n in ("b", "h", "hk", "d", "page"))
    nq, nk = s["seqlen_q"], s["seqlen_k"]
    g = h // hk
    j = torch.arange(nk, device="cuda")
    at = s["table"][:, j // page].clamp(min=0).long()  # [b, keys]
    k = _values(s["k_cache"][at, j % page], s["k_scale"][at, j % page])  # [b, keys, hk, d]
    kt = k.permute(0, 2, 3, 1).contiguous()
    k = None
    v = _values(s["v_cache"][at, j % page], s["v_scale"][at, j % page]).permute(0, 2, 1, 3).contiguous()
    i = torch.arange(nq, device="cuda")
    n = s["cu"][1:] - s["cu"][:-1]
    rows = (s["cu"][:-1, None] + i).clamp(max=s["q"].shape[0] - 1).long()
    q = s["q"][rows].float().view(b, nq, hk, g, d).permute(0, 2, 3, 1, 4).reshape(b, hk, g * nq, d)
    p = torch.matmul(q, kt).mul_(1.0 / math.sqrt(d)).view(b, hk, g, nq, nk)
    last = s["used"][:, None].expand(b, nq)
    if case["causal"]:
        last = torch.minimum(last, s["used"][:, None] - n[:, None] + i[None, :] + 1)
    p.masked_fill_(j >= last[:, None, None, :, None], -math.inf)
    m = p.amax(-1, keepdim=True).clamp(min=-3e38)
    p.sub_(m).exp_()
    z = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(b, hk, g * nq, nk), v).view(b, hk, g, nq, d) / z
    lse = (m + z.log()).squeeze(-1)
    t, seq, _ = _places(s, s["q"].shape[0])
    i = t - s["cu"][seq]
    o = o.permute(0, 3, 1, 2, 4).reshape(b, nq, h, d)[seq, i].to(s["q"].dtype)
    return {"o": o, "lse": lse.reshape(b, h, nq).permute(0, 2, 1)[seq, i].t()}


def _norm(s):
    case, dt = s["case"], s["x"].dtype
    u = s["h"].float()
    if s["w_post"] is not None:
        u = u / (u.square().mean(-1, keepdim=True) + EPS).sqrt() * s["w_post"].float()
    if s["gate"] is not None:
        gate = s["gate"].float()
        u = u * {"none": lambda x: x, "sigmoid": lambda x: 1 / (1 + (-x).exp()), "tanh": torch.tanh}[case["act"]](gate)
    y = s["x"].float() * case["alpha"] + u
    n = y / (y.square().mean(-1, keepdim=True) + EPS).sqrt() * s["w_pre"].float()
    return {"y": y.to(dt), "n": n.to(dt)}


# ---------------------------------------------------------------- one pass
def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        return _norm(s) if op == "norm" else _attend(s) if op == "attend4" else _append(s)
    from compiler_amd import operators as ops
    if op == "norm":
        y, n = ops.block_norm(s["x"], s["h"], s["w_pre"], EPS, w_post=s["w_post"], gate=s["gate"], gate_act=case["act"],
                              residual_scale=case["alpha"])
        return {"y": y, "n": n}
    if op == "attend4":
        o, lse = ops.paged_attention_int4(s["q"], s["k_cache"], s["k_scale"], s["v_cache"], s["v_scale"], s["table"],
                                          s["cu"], s["used"], s["seqlen_q"], s["seqlen_k"], causal=case["causal"])
        return {"o": o, "lse": lse}
    if op == "append":
        q = ops.paged_append(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["k_cache"], s["v_cache"], s["table"],
                             s["cu"], s["used"], interleaved=case["interleaved"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    q, k, v = ops.paged_append_int4(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["k_cache"], s["k_scale"],
                                    s["v_cache"], s["v_scale"], s["table"], s["cu"], s["used"],
                                    interleaved=case["interleaved"], values=True)
    return {"q": q, "k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


# --------------------------------------------------------------------- work
def work(case):
    e, op = SIZE[case["dtype"]], case["op"]
    if op == "norm":
        r, c = case["rows"], case["cols"]
        gate = {"none": 0, "channel": c, "row": r, "full": r * c}[case["gate"]]
        return {"bytes": (4 * r * c + gate + c * (2 if case["post"] else 1)) * e, "flops": 12 * r * c}
    h, hk, d, page = case["h"], case["hk"], case["d"], case["page"]
    ql, kl = _lengths(case)
    t = sum(ql)
    lists = 4 * (2 * case["b"] + 1 + sum((n + page - 1) // page for n in kl))
    if op == "attend4":
        pairs = sum(q * k - (q * (q - 1) // 2 if case["causal"] else 0) for q, k in zip(ql, kl))
        return {"bytes": 2 * t * h * d * e + 4 * h * t + 2 * sum(kl) * hk * (d // 2 + 2 * e) + lists,
                "flops": 4 * h * d * pairs}
    tables = 4 * d * len({k - q + i for q, k in zip(ql, kl) for i in range(q)})
    lists = 4 * (2 * case["b"] + 1 + sum((k - 1) // page - (k - q) // page + 1 for q, k in zip(ql, kl)))
    move = 2 * t * h * d * e + 2 * t * hk * d * e + tables + lists
    # in 4 bits the values that the cache now holds are written beside it
    move += 2 * t * hk * (d * e if op == "append" else d * e + d // 2 + 2 * e)
    return {"bytes": move, "flops": 3 * t * (h + hk) * d + (6 * t * 2 * hk * d if op == "append4" else 0)}


# -------------------------------------------------------------------- exact
def _turned(x, angle, interleaved):
    """Pairs as complex numbers times exp(i angle)."""
    x = x.double()
    half = x.shape[-1] // 2
    pair = x.unflatten(-1, (half, 2)) if interleaved else x.unflatten(-1, (2, half)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * torch.polar(torch.ones_like(angle), angle)[:, None])
    return z.flatten(-2) if interleaved else z.transpose(-1, -2).flatten(-2)


def _held(x, dt):
    """What the 4-bit cache holds of rows x (64 bits): values, scale and offset."""
    lo = x.min(-1, keepdim=True).values
    step = ((x.max(-1, keepdim=True).values - lo) / 15).to(dt).double()
    zero = (lo + 8 * step).to(dt).double()
    level = torch.round((x - zero) / step.clamp(min=2.0 ** -140)).clamp(-8, 7)
    return level * step + zero, torch.cat([step, zero], -1)


def exact(case, seed):
    s = prepare(case, seed)
    op, dt = case["op"], DTYPES[case["dtype"]]
    if op == "norm":
        x, u = s["x"].double(), s["h"].double()
        if s["w_post"] is not None:
            u = u * torch.rsqrt(torch.mean(u ** 2, -1, keepdim=True) + EPS) * s["w_post"].double()
        if s["gate"] is not None:
            z = s["gate"].double()
            u = u * (torch.sigmoid(z) if case["act"] == "sigmoid" else torch.tanh(z) if case["act"] == "tanh" else z)
        y = case["alpha"] * x + u
        return {"y": y, "n": y * torch.rsqrt(torch.mean(y ** 2, -1, keepdim=True) + EPS) * s["w_pre"].double()}
    ql, kl = _lengths(case)
    h, hk, d, page = case["h"], case["hk"], case["d"], case["page"]
    if op == "attend4":
        o = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        lse = torch.empty((h, s["q"].shape[0]), dtype=torch.float64, device="cuda")
        at = 0
        for z, (nq, nk) in enumerate(zip(ql, kl)):
            used = s["table"][z, :(nk + page - 1) // page].long()
            for c in range(hk):
                k, v = ((torch.stack([x[used, :, c] % 16, x[used, :, c] // 16], -1).double().flatten(-2) - 8)
                        * y[used, :, c, :1].double() + y[used, :, c, 1:].double()
                        for x, y in ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"])))
                k, v = (x.reshape(-1, d)[:nk] for x in (k, v))
                heads = slice(c * (h // hk), (c + 1) * (h // hk))
                p = torch.matmul(s["q"][at:at + nq, heads].double().transpose(0, 1).reshape(-1, d), k.t()) / math.sqrt(d)
                p = p.view(-1, nq, nk)
                if case["causal"]:
                    p = p.masked_fill(torch.ones(nq, nk, dtype=torch.bool, device="cuda").triu(nk - nq + 1), -math.inf)
                lse[heads, at:at + nq] = torch.logsumexp(p, -1)
                o[at:at + nq, heads] = (torch.softmax(p, -1).reshape(-1, nk) @ v).view(-1, nq, d).transpose(0, 1)
            at += nq
        return {"o": o, "lse": lse}
    pos = torch.cat([torch.arange(k - q, k) for q, k in zip(ql, kl)]).to("cuda")
    seq = torch.cat([torch.full((q,), z) for z, q in enumerate(ql)]).to("cuda")
    # the tables are inputs: their angle, with the size that their rounding gives them left in
    c, n = s["cos"][pos].double(), s["sin"][pos].double()
    angle, size = torch.atan2(n, c), torch.hypot(n, c)[:, None]
    size = size.repeat_interleave(2, -1) if case["interleaved"] else torch.cat([size, size], -1)
    q, k = (_turned(s[x], angle, case["interleaved"]) * size for x in ("q", "k"))
    v = s["v"].double()
    place = (s["table"][seq, pos // page].long(), pos % page)
    if op == "append":
        kc, vc = (s[x].double() for x in ("k_cache", "v_cache"))
        kc[place], vc[place] = k, v
        return {"q": q, "k_cache": kc, "v_cache": vc}
    (k, ks), (v, vs) = _held(k, dt), _held(v, dt)
    kc, vc = (s[x].double() for x in ("k_scale", "v_scale"))
    kc[place], vc[place] = ks, vs
    return {"q": q, "k": k, "v": v, "k_scale": kc, "v_scale": vc}
