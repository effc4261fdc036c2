"""Paged cache append (16 and 4 bits) and attention over the 4-bit cache on the
GPU, against the float64 oracle.

Tolerances.  Outputs of type T round once: half a step, finfo(T).eps / 2 of the
value.  fp32 rotation adds three roundings of its two products.  4-bit codes,
scales and offsets are defined operation by operation and compare equal.
Attention multiplies codes of at most 8 in magnitude by probability x scale
rounded to bfloat16 (2^-8 of each): 8 x 2^-8 x the largest scale, and half a
step of T; the scores and sums are fp32, whose products run with codes biased by
up to 1032: d x 2^-24 x 1040 x sum |q| x largest scale x softmax scale in the
exponent, which enters O times its spread and LSE as it is.
"""
import math
import threading

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from compiler_amd import operators as ops  # noqa: E402
from compiler_amd import runtime as rt  # noqa: E402
from oracle import paged as ref  # noqa: E402
from own_streams import own_stream  # noqa: E402

pytestmark = pytest.mark.gpu

T = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def dev(x, dt=None):
    t = torch.from_numpy(np.ascontiguousarray(x)).to("cuda")
    return t if dt is None else t.to(T[dt])


def host(t):
    return t.float().cpu().numpy()


def lists(ql, kl, page, rng, spare=2):
    """cu, used, table over shuffled pages, pool size."""
    per = [(n + page - 1) // page for n in kl]
    pool = sum(per) + spare
    order = rng.permutation(pool)
    table = np.full((len(kl), max(per + [1])), -1, np.int32)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    return np.cumsum([0] + list(ql)).astype(np.int32), np.array(kl, np.int32), table, pool


def rope(positions, r, rng):
    a = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(0, r, 2) / max(r, 1))
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


# ------------------------------------------------------------------- append
APPEND = {
    "step": dict(ql=[1, 1, 1], kl=[5, 64, 65], h=8, hk=2, d=128, page=64),
    "one": dict(ql=[1], kl=[1], h=32, hk=8, d=128, page=16),
    "prompt": dict(ql=[70, 1, 133], kl=[70, 40, 140], h=8, hk=2, d=128, page=64),
    "d64_interleaved": dict(ql=[3, 5], kl=[100, 5], h=4, hk=4, d=64, page=16, interleaved=True),
    "interleaved_128": dict(ql=[17, 2], kl=[33, 9], h=4, hk=1, d=128, page=32, interleaved=True),
    "empty_sequences": dict(ql=[0, 4, 0, 0, 2, 0], kl=[9, 4, 0, 7, 30, 1], h=4, hk=2, d=128, page=16),
    "partial": dict(ql=[5, 6], kl=[5, 20], h=4, hk=2, d=128, page=16, r=32),
    "partial_interleaved": dict(ql=[5, 6], kl=[5, 20], h=4, hk=2, d=64, page=16, r=32, interleaved=True),
    "partial_96": dict(ql=[5, 6], kl=[5, 20], h=4, hk=2, d=256, page=16, r=96),
    "partial_16_interleaved": dict(ql=[5, 6], kl=[9, 20], h=4, hk=2, d=32, page=16, r=16, interleaved=True),
    "partial_odd": dict(ql=[5, 6], kl=[5, 20], h=4, hk=2, d=128, page=16, r=26),
    "unturned": dict(ql=[5, 6], kl=[5, 20], h=4, hk=2, d=128, page=16, r=0),
    "odd_d": dict(ql=[4, 3], kl=[4, 11], h=3, hk=3, d=80, page=7),
    "d96": dict(ql=[4, 3], kl=[4, 11], h=6, hk=2, d=96, page=16),
    "d256": dict(ql=[4, 3], kl=[4, 11], h=4, hk=2, d=256, page=32),
    "d32": dict(ql=[9, 3], kl=[9, 11], h=4, hk=2, d=32, page=32),
    "page1": dict(ql=[6, 2], kl=[6, 3], h=4, hk=2, d=64, page=1),
    "many_sequences": dict(ql=[1, 0, 2] * 60, kl=[1 + i for i in range(180)], h=2, hk=1, d=64, page=16),
    "no_queries": dict(ql=[3, 4], kl=[3, 40], h=0, hk=2, d=128, page=16),
    "many_tokens": dict(ql=[1403, 0, 697], kl=[1410, 3, 697], h=43, hk=6, d=128, page=64),  # several groups of heads a wave
}


def append_case(case, dt, seed=0, fused=True):
    c = dict(APPEND[case])
    rng = np.random.default_rng(seed)
    ql, kl, h, hk, d, page = (c[n] for n in ("ql", "kl", "h", "hk", "d", "page"))
    tokens, r = sum(ql), c.get("r", d)
    cu, used, table, pool = lists(ql, kl, page, rng)
    cos, sin = rope(max(kl), r, rng)
    rnd = ref.rounder(dt)
    x = rnd(rng.standard_normal((tokens + 3, h + 2 * hk, d)).astype(np.float32) * 2)  # 3 rows of padding
    return dict(c, interleaved=c.get("interleaved", False), r=r, cu=cu, used=used, table=table, pool=pool, cos=cos, sin=sin,
                q=x[:, :h], k=x[:, h:h + hk], v=x[:, h + hk:], x=x, tokens=tokens)


def turned(c, x):
    pl = ref.places(c["cu"], c["used"], c["table"], x.shape[0], c["page"], c["pool"], len(c["cos"]) if c["r"] else None)
    pos = np.array([p[1] for p in pl])
    cos, sin = (c[n][pos] for n in ("cos", "sin"))
    return pl, ref.rotate(x, cos, sin, c["interleaved"]), ref.rotate(x, cos, sin, c["interleaved"], np.float32)


def close(got, want, dt, extra=0.0, where=""):
    eps = torch.finfo(T[dt]).eps / 2
    tiny = torch.finfo(T[dt]).smallest_normal * torch.finfo(T[dt]).eps
    tol = eps * np.abs(want) + extra + tiny
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (where, int(bad.sum()), float(np.abs(got - want)[bad].max()), np.argwhere(bad)[:3])


def rotation_error(x):
    """Three fp32 roundings of the products and their sum (each pair's |a| + |b| bounds both)."""
    return 3 * 2.0 ** -24 * 2 * np.abs(x).max(-1, keepdims=True)


def append16(c, dt, in_place=False, **kw):
    qkv = dev(c["x"], dt)
    h, hk = c["h"], c["hk"]
    q, k, v = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
    kc = torch.full((c["pool"], c["page"], hk, c["d"]), 9.0, dtype=T[dt], device="cuda")
    vc = kc.clone()
    out = q if in_place else torch.full(q.shape, 9.0, dtype=T[dt], device="cuda")
    ops.paged_append(q, k, v, dev(c["cos"]), dev(c["sin"]), kc, vc, dev(c["table"]), dev(c["cu"]), dev(c["used"]),
                     interleaved=c["interleaved"], out=out, **kw)
    torch.cuda.synchronize()
    return out, kc, vc


def check16(c, dt, out, kc, vc, in_place=False):
    pl, q64, _ = turned(c, c["q"])
    _, k64, _ = turned(c, c["k"])
    want_q = np.full(c["q"].shape, 9.0) if not in_place else c["q"].astype(np.float64)
    want_k = np.full(tuple(kc.shape), 9.0)
    want_v = want_k.copy()
    ek = np.zeros(want_k.shape[:3] + (1,))
    for t, (seq, _, page, row) in enumerate(pl):
        if seq < 0:
            continue
        want_q[t] = q64[t]
        if page >= 0:
            want_k[page, row], want_v[page, row], ek[page, row] = k64[t], c["v"][t], rotation_error(c["k"][t])
    close(host(out), want_q, dt, rotation_error(c["q"]) if c["h"] else 0.0, "q")
    close(host(kc), want_k, dt, ek, "k")
    assert np.array_equal(host(vc), want_v.astype(np.float32))


@pytest.mark.parametrize("dt", sorted(T))
@pytest.mark.parametrize("case", sorted(APPEND))
def test_append(case, dt):
    c = append_case(case, dt)
    check16(c, dt, *append16(c, dt))


@pytest.mark.parametrize("case", ["step", "prompt", "interleaved_128", "partial", "odd_d", "d256"])
def test_append_queries_in_place(case):
    c = append_case(case, "bfloat16")
    check16(c, "bfloat16", *append16(c, "bfloat16", in_place=True), in_place=True)


def append4(c, dt, outs=True):
    h, hk, d = c["h"], c["hk"], c["d"]
    qkv = dev(c["x"], dt)
    q, k, v = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
    kc, ks = ops.int4_cache(c["pool"], c["page"], hk, d, T[dt])
    vc, vs = ops.int4_cache(c["pool"], c["page"], hk, d, T[dt])
    for t in (kc, vc):
        t.fill_(0x5A)
    for t in (ks, vs):
        t.fill_(9.0)
    out = torch.full(q.shape, 9.0, dtype=T[dt], device="cuda")
    ko, vo = (torch.full(k.shape, 9.0, dtype=T[dt], device="cuda") if outs else None for _ in range(2))
    ops.paged_append_int4(q, k, v, dev(c["cos"]), dev(c["sin"]), kc, ks, vc, vs, dev(c["table"]), dev(c["cu"]),
                          dev(c["used"]), interleaved=c["interleaved"], out=out, k_out=ko, v_out=vo)
    torch.cuda.synchronize()
    return out, ko, vo, kc, ks, vc, vs


def check4(c, dt, got):
    out, ko, vo, kc, ks, vc, vs = got
    pl, q64, _ = turned(c, c["q"])
    want_q = np.full(c["q"].shape, 9.0)
    for t, p in enumerate(pl):
        if p[0] >= 0:
            want_q[t] = q64[t]
    close(host(out), want_q, dt, rotation_error(c["q"]) if c["h"] else 0.0, "q")
    for x, turn, codes, scale, vals in ((c["k"], True, kc, ks, ko), (c["v"], False, vc, vs, vo)):
        x32 = turned(c, x)[2] if turn else x.astype(np.float32)
        cd, s, o = ref.quantize(x32, dt)
        want_c = np.full(tuple(codes.shape), 0x5A, np.uint8)
        want_s = np.full(tuple(scale.shape), 9.0, np.float32)
        want_v = np.full(x.shape, 9.0, np.float32)
        for t, (seq, _, page, row) in enumerate(pl):
            if seq < 0:
                continue
            want_v[t] = ref.rounder(dt)(((cd[t].astype(np.float64) - 8) * s[t] + o[t]).astype(np.float32))
            if page >= 0:
                want_c[page, row] = ref.pack(cd[t])
                want_s[page, row] = np.concatenate([s[t], o[t]], -1)
        assert np.array_equal(codes.cpu().numpy(), want_c)
        assert np.array_equal(host(scale), want_s, equal_nan=True)
        if vals is not None:
            assert np.array_equal(host(vals), want_v, equal_nan=True)


@pytest.mark.parametrize("dt", ["bfloat16", "float16"])
@pytest.mark.parametrize("case", sorted(APPEND))
def test_append_int4(case, dt):
    c = append_case(case, dt)
    got = append4(c, dt)
    check4(c, dt, got)
    bare = append4(c, dt, outs=False)
    for a, b in zip(got[3:], bare[3:]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dt", ["bfloat16", "float16"])
@pytest.mark.parametrize("case", ["prompt", "odd_d", "d64_interleaved"])
def test_append_int4_special_rows(case, dt):
    """Rows of one value, of zeros, with the type's extremes, tiny, with inf and NaN."""
    c = append_case(case, dt)
    big = float(torch.finfo(T[dt]).max)
    v = c["v"]
    v[0] = 0.0
    v[1] = 3.0
    v[2, 0], v[2, 0, 3] = 1.0, big
    v[3, 0], v[3, 0, :2] = 0.0, (big, -big)
    v[4, 0, 5] = np.inf
    v[5, 0, 7] = np.nan
    v[6] = v[6] * (2.0 ** -130 if dt == "bfloat16" else 2.0 ** -24)
    c["x"][:, c["h"] + c["hk"]:] = ref.rounder(dt)(v)
    c["v"] = c["x"][:, c["h"] + c["hk"]:]
    check4(c, dt, append4(c, dt))


def test_append_bad_places():
    """Pages outside the pool and the table, positions below 0 and past the
    cos / sin tables, sequences outside the tokens: left out, the rest done."""
    for dt, four in (("bfloat16", False), ("bfloat16", True), ("float32", False)):
        c = append_case("prompt", dt)
        c["table"][0, 0], c["table"][2, 1] = -3, c["pool"]
        c["table"] = c["table"][:, :2]          # sequence 2's third page is not in the table
        c["cos"], c["sin"] = c["cos"][:139], c["sin"][:139]
        c["used"][1] = 0                        # position -1
        check4(c, dt, append4(c, dt)) if four else check16(c, dt, *append16(c, dt))
        c["cu"][3] = c["x"].shape[0] + 1        # past the tokens
        check4(c, dt, append4(c, dt)) if four else check16(c, dt, *append16(c, dt))
        c["cu"][:] = [5, 2, -7, 1 << 30]        # no sequence at all
        check4(c, dt, append4(c, dt)) if four else check16(c, dt, *append16(c, dt))


def test_append_strides_and_16_bit_tables():
    """Head-major inputs, a padded cache with its own strides, tables in the model's type."""
    dt = "bfloat16"
    for case in ("prompt", "odd_d"):
        c = append_case(case, dt)
        rnd = ref.rounder(dt)
        c["cos"], c["sin"] = rnd(c["cos"]), rnd(c["sin"])
        h, hk, d = c["h"], c["hk"], c["d"]
        hm = dev(c["x"].transpose(1, 0, 2), dt).transpose(0, 1)
        pool = torch.full((hk, c["pool"], c["page"] + 1, d + 6), 9.0, dtype=T[dt], device="cuda")
        kc = pool[:, :, :c["page"], :d].permute(1, 2, 0, 3)
        vc = pool.clone()[:, :, :c["page"], :d].permute(1, 2, 0, 3)
        out = torch.full((h, c["x"].shape[0], d), 9.0, dtype=T[dt], device="cuda").transpose(0, 1)
        ops.paged_append(hm[:, :h], hm[:, h:h + hk], hm[:, h + hk:], dev(c["cos"], dt), dev(c["sin"], dt), kc, vc,
                         dev(c["table"]), dev(c["cu"]), dev(c["used"]), out=out, sync=True)
        check16(c, dt, out, kc, vc)
        assert (pool[:, :, c["page"]:] == 9.0).all() and (pool[..., d:] == 9.0).all()


# ---------------------------------------------------------------- attention
ATTEND = {
    "one_key": dict(ql=[1], kl=[1], h=4, hk=4, d=128, page=64),
    "tile_edges": dict(ql=[1, 1, 1, 1], kl=[15, 16, 17, 33], h=8, hk=2, d=128, page=16),
    "round_edges": dict(ql=[1, 1, 1], kl=[127, 128, 129], h=8, hk=1, d=64, page=64),
    "ranges": dict(ql=[1, 1], kl=[1500, 700], h=32, hk=8, d=128, page=64),
    "ranges_d64": dict(ql=[2, 1], kl=[2051, 300], h=16, hk=4, d=64, page=16),
    "d256": dict(ql=[1, 2], kl=[600, 77], h=8, hk=2, d=256, page=32),
    "rows32": dict(ql=[4, 3], kl=[700, 300], h=8, hk=1, d=128, page=16),
    "rows17": dict(ql=[17], kl=[513], h=2, hk=2, d=64, page=16),
    "rows33": dict(ql=[33, 5], kl=[300, 40], h=2, hk=2, d=128, page=16),
    "chunk": dict(ql=[130, 64, 1], kl=[500, 64, 3], h=8, hk=2, d=128, page=64),
    "chunk_d64": dict(ql=[90, 7], kl=[260, 300], h=6, hk=2, d=64, page=32),
    "group3": dict(ql=[5, 2], kl=[300, 2], h=6, hk=2, d=128, page=16),
    "noncausal": dict(ql=[5, 20], kl=[200, 20], h=4, hk=2, d=128, page=16, causal=False),
    "local": dict(ql=[4, 1], kl=[900, 80], h=4, hk=2, d=128, page=16, window=(100, 0)),
    "local_both": dict(ql=[40, 9], kl=[400, 9], h=4, hk=2, d=64, page=64, causal=False, window=(30, 7)),
    "fewer_keys_than_queries": dict(ql=[8, 3], kl=[5, 1], h=2, hk=1, d=64, page=16),
    "no_keys_no_queries": dict(ql=[3, 0, 2, 1], kl=[0, 40, 2, 500], h=4, hk=2, d=128, page=16),
    "page48": dict(ql=[1, 2], kl=[400, 100], h=4, hk=4, d=128, page=48),
    "page1": dict(ql=[1, 2], kl=[70, 9], h=4, hk=2, d=64, page=1),
    "page10": dict(ql=[1, 2], kl=[170, 9], h=4, hk=2, d=128, page=10),
    "wide": dict(ql=[1] * 32, kl=[1 + 37 * i for i in range(32)], h=16, hk=8, d=128, page=16),
    "wide_d64": dict(ql=[1, 0, 1, 2] * 8, kl=[1100 - 31 * i for i in range(32)], h=8, hk=8, d=64, page=64),
    "wide_few": dict(ql=[3, 1, 2, 0], kl=[1024, 513, 30, 700], h=8, hk=2, d=128, page=16),
    "wide_few_d64": dict(ql=[2, 5], kl=[2, 1000], h=6, hk=2, d=64, page=32, causal=False, window=(511, 2)),
    "odd_d": dict(ql=[2, 1], kl=[70, 300], h=4, hk=2, d=80, page=16),
    "d2": dict(ql=[2], kl=[70], h=2, hk=1, d=2, page=16),
}


def attend_case(case, dt, seed=0):
    c = dict(ATTEND[case]) if isinstance(case, str) else dict(case)
    rng = np.random.default_rng(seed)
    ql, kl, h, hk, d, page = (c[n] for n in ("ql", "kl", "h", "hk", "d", "page"))
    cu, used, table, pool = lists(ql, kl, page, rng)
    rnd = ref.rounder(dt)
    c.update(cu=cu, used=used, table=table, pool=pool, causal=c.get("causal", True), window=c.get("window", (-1, -1)),
             q=rnd(rng.standard_normal((sum(ql) + 3, h, d)).astype(np.float32)),
             seqlen_q=max(ql), seqlen_k=max(kl), scale=c.get("scale", 1 / math.sqrt(d)))
    for n in ("k", "v"):
        x = rng.standard_normal((pool, page, hk, d)).astype(np.float32)
        if n == "k":
            x[..., 1] += 4.0  # an off-centre channel
        cd, s, o = ref.quantize(x, dt)
        c[n + "c"], c[n + "s"] = ref.pack(cd), np.concatenate([s, o], -1)
    return c


def head_major(x, dt=None):
    return dev(x.transpose(0, 2, 1, 3), dt).transpose(1, 2)


def attend_args(c, dt):
    return (dev(c["q"], dt), head_major(c["kc"]), head_major(c["ks"], dt), head_major(c["vc"]), head_major(c["vs"], dt),
            dev(c["table"]), dev(c["cu"]), dev(c["used"]), c["seqlen_q"], c["seqlen_k"])


def attend_run(c, dt, args=None, **kw):
    args = attend_args(c, dt) if args is None else args
    o = torch.full(c["q"].shape, 9.0, dtype=T[dt], device="cuda")
    lse = torch.full((c["h"], c["q"].shape[0]), 9.0, device="cuda")
    ops.paged_attention_int4(*args, scale=c["scale"], causal=c["causal"], window=c["window"], out=o, lse=lse, **kw)
    torch.cuda.synchronize()
    return o, lse


def attend_want(c):
    keys = {"k": [], "v": []}
    seen = []
    for b, n in enumerate(c["used"]):
        j = np.arange(max(0, min(int(n), c["table"].shape[1] * c["page"])))
        at = c["table"][b, j // c["page"]]
        seen.append((at >= 0) & (at < c["pool"]))
        at = np.where(seen[-1], at, 0)
        for x in ("k", "v"):
            keys[x].append(ref.values(c[x + "c"][at, j % c["page"]], c[x + "s"][at, j % c["page"]]))
    right = 0 if c["causal"] else c["window"][1]
    return ref.attention(c["q"], keys["k"], keys["v"], c["used"], c["cu"], c["scale"], c["window"][0], right,
                         c["seqlen_q"], seen)


def check_attend(c, dt, o, lse):
    wo, wl, rows = attend_want(c)
    fine = np.nan_to_num(c["ks"]), np.nan_to_num(c["vs"])
    score = c["d"] * 2.0 ** -24 * 1040 * np.abs(c["q"]).sum(-1).max(initial=0) * np.abs(fine[0]).max() * abs(c["scale"])
    extra = 8 * 2.0 ** -8 * np.abs(fine[1][..., 0]).max() + 2 * score * np.abs(wo).max(initial=0)
    go, gl = host(o), lse.cpu().numpy()
    close(go[rows], wo[rows], dt, extra, "o")
    assert (go[~rows] == 9.0).all() and (gl[:, ~rows] == 9.0).all()
    gl, wl = gl[:, rows], wl[:, rows]
    assert np.array_equal(np.isinf(gl), np.isinf(wl))
    f = np.isfinite(wl)
    err = np.abs(gl[f] - wl[f])
    assert (err <= score + 2.0 ** -20 * (1 + np.abs(wl[f]))).all(), float(err.max())


# the form that a case takes where it has one of its own to show
FORMS = {"one_key": "_r1", "ranges": "_r1_merge", "rows32": "_r2", "d256": "_r1", "wide": "_r1w", "wide_d64": "_r1w",
         "wide_few": "_r1w", "wide_few_d64": "_r1w", "local": "_r1w",
         "chunk": "_r2", "page1": "_general", "page10": "_general", "odd_d": "_general", "d2": "_general"}


@pytest.mark.parametrize("dt", ["bfloat16", "float16"])
@pytest.mark.parametrize("case", sorted(ATTEND))
def test_attend(case, dt):
    c = attend_case(case, dt)
    check_attend(c, dt, *attend_run(c, dt))
    assert rt.module().last_kernel.endswith(FORMS.get(case, ""))


def test_attend_scores_climb():
    """Every tile moves the running maximum, by about 16 log2 units a tile."""
    c = attend_case(dict(ql=[1, 3], kl=[2000, 900], h=8, hk=2, d=128, page=64), "bfloat16")
    x = ref.values(c["kc"], c["ks"]).astype(np.float32)
    for b, n in enumerate(c["used"]):
        j = np.arange(int(n))
        x[c["table"][b, j // 64], j % 64, :, 0] = (j / 8.0)[:, None]
    cd, s, o = ref.quantize(x, "bfloat16")
    c["kc"], c["ks"] = ref.pack(cd), np.concatenate([s, o], -1)
    c["q"][..., 0] = 4.0
    check_attend(c, "bfloat16", *attend_run(c, "bfloat16"))


@pytest.mark.parametrize("case", ["ranges", "chunk", "odd_d", "local", "wide_few", "wide_few_d64"])
def test_attend_nothing_leaks_from_unseen_places(case):
    """NaN scales in every cache row that no query sees: behind the sequences'
    ends, in unused pages, and (for the causal queries) after them."""
    c = attend_case(case, "bfloat16")
    want = [x.clone() for x in attend_run(c, "bfloat16")]
    used = np.zeros((c["pool"], c["page"]), bool)
    for b, n in enumerate(c["used"]):
        j = np.arange(int(n))
        used[c["table"][b, j // c["page"]], j % c["page"]] = True
    for n in ("ks", "vs"):
        c[n][~used] = np.nan
    got = attend_run(c, "bfloat16")
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    check_attend(c, "bfloat16", *got)


def test_attend_nan_after_a_query_stays_there():
    """A NaN key and value that only the later queries see leaves the earlier ones alone."""
    c = attend_case("chunk", "bfloat16")
    want = [x.clone() for x in attend_run(c, "bfloat16")]
    j = 460  # sequence 0 holds 500 keys, its queries stand at 370 .. 499
    c["ks"][c["table"][0, j // 64], j % 64] = np.nan
    c["vs"][c["table"][0, j // 64], j % 64] = np.nan
    o, lse = attend_run(c, "bfloat16")
    assert torch.equal(o[:90], want[0][:90]) and torch.equal(lse[:, :90], want[1][:, :90])
    assert torch.equal(o[130:], want[0][130:])
    assert torch.isnan(o[90:130]).all()


@pytest.mark.parametrize("case", ["ranges", "chunk", "rows17", "wide_few", "odd_d", "d256"])
def test_attend_bad_query_rows_stay_alone(case):
    """NaN or infinities in one query row (one head of one token) leave the others' bits."""
    c = attend_case(case, "bfloat16")
    want = [x.clone() for x in attend_run(c, "bfloat16")]
    t, h = 1, c["h"] - 1
    keep = torch.ones(c["q"].shape[:2], dtype=torch.bool, device="cuda")
    keep[t, h] = False
    for bad in (np.nan, np.inf, -np.inf):
        c["q"][t, h, 5] = bad
        o, lse = attend_run(c, "bfloat16")
        assert torch.equal(o[keep], want[0][keep]) and torch.equal(lse.t()[keep], want[1].t()[keep])
        assert torch.isnan(o[t, h]).all()


@pytest.mark.parametrize("case", ["ranges", "chunk", "odd_d", "page10", "d256", "wide_few"])
def test_attend_bad_pages_count_as_no_keys(case):
    c = attend_case(case, "bfloat16")
    c["table"][0, 0], c["table"][0, -1], c["table"][-1, 0] = -1, c["pool"], 1 << 30
    check_attend(c, "bfloat16", *attend_run(c, "bfloat16"))
    c["used"][0] = c["table"].shape[1] * c["page"] + 1000  # more keys than the table names
    check_attend(c, "bfloat16", *attend_run(c, "bfloat16"))
    c["cu"][-1] = c["q"].shape[0] + 1                      # a sequence outside q
    check_attend(c, "bfloat16", *attend_run(c, "bfloat16"))
    c["used"][:] = -5
    check_attend(c, "bfloat16", *attend_run(c, "bfloat16"))


@pytest.mark.parametrize("case", ["ranges", "rows33", "odd_d"])
def test_attend_queries_past_seqlen_q_are_left_alone(case):
    c = attend_case(case, "bfloat16")
    c["seqlen_q"] = max(1, c["seqlen_q"] // 2)
    c["seqlen_k"] = 100  # only shapes the key ranges
    check_attend(c, "bfloat16", *attend_run(c, "bfloat16"))


def test_attend_other_layouts():
    """Token-major pages, padded rows, head-major queries, a strided lse."""
    c = attend_case("ranges", "float16")
    a = list(attend_args(c, "float16"))
    a[0] = a[0].transpose(0, 1).contiguous().transpose(0, 1)
    for i in (1, 3):
        pad = torch.zeros(a[i].shape[:3] + (a[i].shape[3] + 16,), dtype=torch.uint8, device="cuda")
        pad[..., :a[i].shape[3]] = a[i]
        a[i] = pad[..., :a[i].shape[3]]
    for i in (2, 4):
        a[i] = a[i].contiguous()
    o = torch.full(c["q"].shape, 9.0, dtype=torch.float16, device="cuda").transpose(0, 1).contiguous().transpose(0, 1)
    lse = torch.full((c["q"].shape[0], c["h"]), 9.0, device="cuda").t()
    ops.paged_attention_int4(*a, scale=c["scale"], out=o, lse=lse, sync=True)
    check_attend(c, "float16", o, lse)
    # codes that are not 16-byte aligned
    flat = torch.zeros(a[1].numel() + 3, dtype=torch.uint8, device="cuda")
    a[1] = flat[3:].view(a[1].shape).copy_(a[1])
    o.fill_(9.0)
    lse.fill_(9.0)
    ops.paged_attention_int4(*a, scale=c["scale"], out=o, lse=lse, sync=True)
    check_attend(c, "float16", o, lse)


# ------------------------------------------------------- a step, run together
def test_append_then_attend_steps():
    """A prompt chunk and decoding steps through the cache: the attention sees
    exactly what the appends say they hold; also from a captured graph, replayed
    between the program's own work, and on another stream."""
    dt, h, hk, d, page, b = torch.bfloat16, 8, 2, 128, 16, 3
    rng = np.random.default_rng(5)
    room = 12
    table = dev(rng.permutation(b * room).reshape(b, room).astype(np.int32))
    kc, ks = ops.int4_cache(b * room, page, hk, d, dt)
    vc, vs = ops.int4_cache(b * room, page, hk, d, dt)
    cos, sin = (dev(x) for x in rope(room * page, d, rng))
    held = [[], []], [[], []], [[], []]

    def want(i, q, n):
        k, v = (torch.cat(x).double() for x in held[i])
        k, v = (x.repeat_interleave(h // hk, 1) for x in (k, v))
        s = torch.einsum("qhd,khd->hqk", q.double().cpu(), k) / math.sqrt(d)
        keys = k.shape[0]
        mask = torch.arange(keys)[None, :] > torch.arange(n)[:, None] + keys - n
        s.masked_fill_(mask[None], -math.inf)
        return torch.einsum("hqk,khd->qhd", torch.softmax(s, -1), v)

    lens = np.zeros(b, np.int64)
    graph = None
    for step in range(5):
        ql = [[70, 33, 1]] + [[1, 1, 1]] * 4
        n = ql[step]
        cu = dev(np.cumsum([0] + n).astype(np.int32))
        lens += n
        used = dev(lens.astype(np.int32))
        qkv = torch.randn(sum(n), h + 2 * hk, d, device="cuda").to(dt)
        q, k, v = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]

        def call():
            qr, kv, vv = ops.paged_append_int4(q, k, v, cos, sin, kc, ks, vc, vs, table, cu, used, values=True)
            o, _ = ops.paged_attention_int4(qr, kc, ks, vc, vs, table, cu, used, max(n), int(lens.max()))
            return qr, kv, vv, o
        if step == 2:
            stream = own_stream()
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                out = call()
            stream.synchronize()
        elif step == 3:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=own_stream()):
                out = call()
            first = None
            for _ in range(3):
                for x in out:
                    x.zero_()
                torch.cuda.synchronize()
                graph.replay()
                torch.cuda.synchronize()
                now = [x.clone() for x in out]
                assert first is None or all(torch.equal(x, y) for x, y in zip(now, first))
                first = now
                assert all(torch.equal(x, y) for x, y in zip(call(), now))
        else:
            out = call()
        torch.cuda.synchronize()
        qr, kv, vv, o = (x.cpu() for x in out)
        at = 0
        for i in range(b):
            held[i][0].append(kv[at:at + n[i]])
            held[i][1].append(vv[at:at + n[i]])
            w = want(i, qr[at:at + n[i]], n[i])
            # the held values round to bf16 (2^-8 of up to 8 scales, scores by as much of the
            # keys); the bars of the 16-bit kernels
            assert torch.allclose(o[at:at + n[i]].double(), w, rtol=2e-2, atol=4e-2)
            at += n[i]


@pytest.mark.parametrize("case", ["ranges", "rows32", "d256", "ranges_d64"])
def test_attend_workspace_may_hold_anything(case):
    """The records of parts that a shorter sequence does not have count for nothing."""
    c = attend_case(case, "bfloat16")
    c["seqlen_k"] = 4096  # more parts than any sequence has
    args = attend_args(c, "bfloat16")
    size = rt.module().attention_int4_workspace(len(c["used"]), c["h"], c["hk"], c["d"], c["seqlen_q"], 4096)
    got = []
    for fill in (0.0, math.nan, math.inf):
        got.append(attend_run(c, "bfloat16", args, workspace=torch.full((size,), fill, device="cuda")))
        assert rt.module().last_kernel.endswith("_merge")
    assert all(torch.equal(a, b) for g in got[1:] for a, b in zip(g, got[0]))
    check_attend(c, "bfloat16", *got[0])


def test_attend_parts_in_captured_graphs():
    """Calls of several parts captured into two graphs (each with its own workspace,
    from torch's allocator): replayed in turn, between eager calls of other
    sizes, each gives its eager bits again."""
    cases = [attend_case("ranges", "bfloat16"), attend_case("rows32", "bfloat16", seed=3)]
    cases[1]["seqlen_k"] = 2000  # several parts
    args = [attend_args(c, "bfloat16") for c in cases]
    call = lambda i: ops.paged_attention_int4(*args[i], scale=cases[i]["scale"])  # noqa: E731
    want = []
    for i, c in enumerate(cases):
        want.append([x.clone() for x in call(i)])
        assert rt.module().last_kernel.endswith("_merge")
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=own_stream()):
            outs.append(call(i))
        graphs.append(g)
    for _ in range(3):
        for i in (0, 1):
            for x in outs[i]:
                x.zero_()
            torch.cuda.synchronize()
            graphs[i].replay()
            ops.paged_attention_int4(*args[1 - i], scale=cases[1 - i]["scale"])
            torch.cuda.synchronize()
            n = cases[i]["q"].shape[0] - 3
            assert torch.equal(outs[i][0][:n], want[i][0][:n]) and torch.equal(outs[i][1][:, :n], want[i][1][:, :n])


def test_attend_streams_workspaces_and_prepared_calls():
    """A Stream, its handle, the per-thread stream (which gets no workspace), a given
    workspace of any length, a prepared call."""
    c = attend_case("ranges", "bfloat16")
    args = attend_args(c, "bfloat16")
    n = c["q"].shape[0] - 3
    side = own_stream()
    torch.cuda.synchronize()
    for stream in (side, side.cuda_stream, 0, 2):
        o, lse = ops.paged_attention_int4(*args, scale=c["scale"], stream=stream, sync=True)
        assert rt.module().last_kernel.endswith("_merge") == (stream != 2)
        check_attend(c, "bfloat16", torch.cat([o[:n], torch.full_like(o[n:], 9)]),
                     torch.cat([lse[:, :n], torch.full_like(lse[:, n:], 9)], 1))
    need = rt.module().attention_int4_workspace(2, 32, 8, 128, 1, 1500)
    assert need > 0
    for floats in (0, 7, need // 2, need, need + 99):
        o, lse = attend_run(c, "bfloat16", args, workspace=torch.empty(floats, device="cuda"))
        assert rt.module().last_kernel.endswith("_merge") == (floats >= need // 2)
        check_attend(c, "bfloat16", o, lse)
    with pytest.raises(rt.G950Error, match="16-byte aligned"):
        attend_run(c, "bfloat16", args, workspace=torch.empty(need + 1, device="cuda")[1:])
    o = torch.full(c["q"].shape, 9.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((c["h"], n + 3), 9.0, device="cuda")
    call = ops.paged_attention_int4_kernel(*args[:8], o, lse, torch.empty(need, device="cuda"), c["seqlen_q"], c["seqlen_k"],
                                           c["scale"], True, -1, -1, prepare=True)
    for _ in range(2):
        call()
    torch.cuda.synchronize()
    check_attend(c, "bfloat16", o, lse)


@pytest.mark.parametrize("d,dt", [(128, "bfloat16"), (64, "float16"), (80, "bfloat16")])
def test_caches_past_32_bits(d, dt):
    """Pages more than 2^31 (and 2^32) elements apart: append and attention by the
    fast kernels and the general one."""
    far = 3 << 30
    rng = np.random.default_rng(3)
    cu, used = np.array([0, 3, 4], np.int32), np.array([40, 17], np.int32)
    table = np.array([[1, 0, 2], [3, 4, -1]], np.int32)
    rows = 16 * 2 * (d // 2)
    raw = [torch.zeros(4 * far + rows, dtype=torch.uint8, device="cuda") for _ in range(2)]
    codes = [x.as_strided((5, 16, 2, d // 2), (far, d, d // 2, 1)) for x in raw]
    scales = [torch.zeros((5, 2, 16, 2), dtype=T[dt], device="cuda").transpose(1, 2) for _ in range(2)]
    cos, sin = rope(40, d, rng)
    rnd = ref.rounder(dt)
    ks, vs = [], []
    # the whole sequences appended as one prompt, then the last tokens attend
    x = rnd(rng.standard_normal((57, 8, d)).astype(np.float32))
    full = dev(np.array([0, 40, 57], np.int32))
    q, kv, vv = ops.paged_append_int4(dev(x[:, :4], dt), dev(x[:, 4:6], dt), dev(x[:, 6:], dt), dev(cos), dev(sin), codes[0],
                                      scales[0], codes[1], scales[1], dev(table), full, dev(used), values=True)
    name = rt.module().last_kernel
    assert name.endswith("general" if d == 80 else f"d{d}")
    pick = [37, 38, 39, 56]
    o, lse = ops.paged_attention_int4(q[pick].contiguous(), codes[0], scales[0], codes[1], scales[1], dev(table), dev(cu),
                                      dev(used), 3, 40, sync=True)
    assert rt.module().last_kernel.endswith("general" if d == 80 else "_r1")
    for lo, hi in ((0, 40), (40, 57)):
        ks.append(host(kv)[lo:hi].astype(np.float64))
        vs.append(host(vv)[lo:hi].astype(np.float64))
    wo, wl, _ = ref.attention(host(q)[pick], ks, vs, used, cu, 1 / math.sqrt(d), -1, 0, 3)
    # the values that came back are rounded to 16 bits (2^-8 of up to 4.5 in keys and values)
    assert np.abs(host(o) - wo).max() < 0.06 and np.abs(lse.cpu().numpy() - wl).max() < 0.06
    # 16 bits
    kc = torch.zeros(2 * far + 16 * 2 * d, dtype=T[dt], device="cuda").as_strided((3, 16, 2, d), (far, 2 * d, d, 1))
    vc = torch.zeros((3, 16, 2, d), dtype=T[dt], device="cuda")
    ops.paged_append(None, dev(x[:40, 4:6], dt), dev(x[:40, 6:], dt), dev(cos), dev(sin), kc, vc, dev(table[:1] % 3),
                     dev(np.array([0, 40], np.int32)), dev(used[:1]), sync=True)
    c1, s1 = cos[:40], sin[:40]
    want = ref.rotate(x[:40, 4:6], c1, s1, False)
    got = np.concatenate([host(kc[int(p) % 3]) for p in table[0]])[:40]
    close(got, want, dt, rotation_error(x[:40, 4:6]))


def test_no_sequences():
    """b = 0: nothing is read or written, whatever the other extents."""
    e = torch.empty((0, 3), dtype=torch.int32, device="cuda")
    cu, used = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda")
    for tokens in (0, 2):
        q = torch.randn(tokens, 4, 128, device="cuda").bfloat16()
        kc, ks = ops.int4_cache(2, 16, 2, 128, torch.bfloat16)
        out = torch.full_like(q, 9.0)
        cos = torch.ones(4, 64, device="cuda")
        ops.paged_append_int4(q, q[:, :2], q[:, 2:], cos, cos, kc, ks, kc.clone(), ks.clone(), e, cu, used, out=out)
        o, lse = ops.paged_attention_int4(q, kc, ks, kc, ks, e, cu, used, 1, 16, out=out, sync=True)
        assert (out == 9.0).all() and (kc == 0).all() and o is out


def test_other_calls_are_refused():
    c = append_case("step", "bfloat16")
    q = dev(c["q"], "bfloat16")
    with pytest.raises(rt.G950Error, match="current device"):
        ops.paged_append(q.cpu(), q[:, :2], q[:, :2], dev(c["cos"]), dev(c["sin"]), q, q, dev(c["table"]), dev(c["cu"]),
                         dev(c["used"]))
    with pytest.raises(rt.G950Error, match="be the input"):
        kc, ks = ops.int4_cache(c["pool"], 64, 2, 128, torch.bfloat16)
        k = q[:, :2]
        ops.paged_append_int4(q, k, k, dev(c["cos"]), dev(c["sin"]), kc, ks, kc.clone(), ks.clone(), dev(c["table"]),
                              dev(c["cu"]), dev(c["used"]), k_out=k, v_out=torch.empty_like(k))


def test_append_int4_one_of_the_values():
    c = append_case("prompt", "bfloat16")
    both = append4(c, "bfloat16")
    qkv = dev(c["x"], "bfloat16")
    h, hk = c["h"], c["hk"]
    for name, want in (("k_out", both[1]), ("v_out", both[2])):
        kc, ks = ops.int4_cache(c["pool"], c["page"], hk, c["d"], torch.bfloat16)
        out = torch.full(want.shape, 9.0, dtype=torch.bfloat16, device="cuda")
        _, ko, vo = ops.paged_append_int4(qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:], dev(c["cos"]), dev(c["sin"]), kc, ks,
                                          kc.clone(), ks.clone(), dev(c["table"]), dev(c["cu"]), dev(c["used"]), sync=True,
                                          **{name: out})
        assert (ko is None) == (name == "v_out") and (vo is None) == (name == "k_out")
        assert torch.equal(out, want)


def test_calls_from_two_threads_on_two_streams():
    c = attend_case("ranges", "bfloat16")
    args = attend_args(c, "bfloat16")
    want = [x.clone() for x in attend_run(c, "bfloat16", args)]
    bad = []

    def work(i):
        s = own_stream(i)
        with torch.cuda.stream(s):
            for _ in range(20):
                o, lse = ops.paged_attention_int4(*args, scale=c["scale"])
                s.synchronize()
                n = c["q"].shape[0] - 3
                if not (torch.equal(o[:n], want[0][:n]) and torch.equal(lse[:, :n], want[1][:, :n])):
                    bad.append(1)
    own_stream(0), own_stream(1)
    th = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in th:
        t.start()
    for t in th:
        t.join()
    assert not bad


def test_no_alloc_calls():
    c = append_case("prompt", "bfloat16")
    with rt.no_alloc():
        check16(c, "bfloat16", *append16(c, "bfloat16"))
        check4(c, "bfloat16", append4(c, "bfloat16"))
        a = attend_case("ranges", "bfloat16")
        check_attend(a, "bfloat16", *attend_run(a, "bfloat16"))
