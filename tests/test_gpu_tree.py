"""Drafted token trees on the GPU against the float64 oracle: append, attention,
verification, the move of the accepted rows, and a step of all four.

Attention's bars (u = 2^-24, half a step of fp32; U = 2^-23 for sums inside the matrix
cores, whose rounding is not documented; h = finfo(T).eps / 2):
  * a score is d exact products (fp32 models: rounded ones) summed in fp32: U d sum |q k| scale; scale in
    log2 units, the exponent's product and subtraction, exp2: 6 u |s| + 2^-22.  e: their sum's largest.
  * LSE: e, and 2^-20 (1 + |LSE| / 2) for its sum and log.
  * O: 2 e sum p |V| from the scores; a probability rounds to T (h of itself; below float16's
    normals 2^-25 of the largest; not in fp32 models): h sum p |V| (+ 2^-25 sum |V| / l); sums of m
    keys, weights joined: U (m + 64) sum p |V|; O rounds once: h |O|.
"""
import math
import threading

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from compiler_amd import operators as ops  # noqa: E402
from compiler_amd import runtime as rt  # noqa: E402
from oracle import paged, tree as ref  # noqa: E402
from own_streams import own_stream  # noqa: E402
from test_gpu_paged_int4 import T, close, dev, host, lists, rope, rotation_error  # noqa: E402

pytestmark = pytest.mark.gpu

U = 2.0 ** -23


def tree_of(kind, n, rng):
    """Parents of n nodes."""
    if kind == "chain":
        return [i - 1 for i in range(n)]
    if kind == "star":
        return [-1] + [0] * (n - 1)
    if kind == "forest":  # any parent or none, some of them no node before the own
        return [int(rng.integers(-2, n + 1)) for _ in range(n)]
    return [-1] + [int(rng.integers(max(0, i // 3 - 2), i)) for i in range(1, n)][:n - 1] if n else []


def forest(c, rng):
    kinds = c.get("kinds", ["tree"])
    return np.array([x for z, n in enumerate(c["ql"]) for x in tree_of(kinds[z % len(kinds)], n, rng)] + [0] * 3, np.int32)


# ------------------------------------------------------------------- append
APPEND = {
    "one": dict(ql=[1], kl=[1], h=32, hk=8, d=128, page=16),
    "trees": dict(ql=[26, 1, 9], kl=[90, 40, 9], h=8, hk=2, d=128, page=64),
    "interleaved": dict(ql=[13, 5], kl=[100, 5], h=4, hk=4, d=64, page=16, interleaved=True),
    "chain": dict(ql=[70, 3], kl=[70, 20], h=4, hk=2, d=128, page=16, kinds=["chain"]),
    "deep_tree": dict(ql=[200, 130], kl=[300, 130], h=4, hk=1, d=32, page=32),
    "forest": dict(ql=[64, 65, 7], kl=[64, 100, 30], h=2, hk=2, d=256, page=16, kinds=["forest"]),
    "star": dict(ql=[40], kl=[50], h=4, hk=2, d=64, page=16, kinds=["star"]),
    "empty_sequences": dict(ql=[0, 4, 0, 0, 2, 0], kl=[9, 4, 0, 7, 30, 1], h=4, hk=2, d=128, page=16),
    "partial": dict(ql=[15, 6], kl=[15, 20], h=4, hk=2, d=128, page=16, r=32),
    "odd_d": dict(ql=[14, 3], kl=[14, 11], h=3, hk=3, d=80, page=7),
    "no_queries": dict(ql=[13, 4], kl=[13, 40], h=0, hk=2, d=128, page=16),
    "many": dict(ql=[30] * 70, kl=[31 + i for i in range(70)], h=8, hk=2, d=64, page=16),
}


def append_case(name, dt, seed=0):
    c = dict(APPEND[name])
    rng = np.random.default_rng(seed)
    r, tokens = c.get("r", c["d"]), sum(c["ql"])
    cu, used, table, pool = lists(c["ql"], c["kl"], c["page"], rng)
    cos, sin = rope(max(c["kl"]), r, rng)
    x = paged.rounder(dt)(rng.standard_normal((tokens + 3, c["h"] + 2 * c["hk"], c["d"])).astype(np.float32) * 2)
    c.update(interleaved=c.get("interleaved", False), r=r, cu=cu, used=used, table=table, pool=pool, cos=cos, sin=sin, x=x,
             parent=forest(c, rng))
    return c


def append_run(c, dt, in_place=False, **kw):
    x, h, hk = dev(c["x"], dt), c["h"], c["hk"]
    q, k, v = x[:, :h], x[:, h:h + hk], x[:, h + hk:]
    kc = torch.full((c["pool"], c["page"], hk, c["d"]), 9.0, dtype=T[dt], device="cuda")
    vc = kc.clone()
    out = q if in_place else torch.full(q.shape, 9.0, dtype=T[dt], device="cuda")
    ops.paged_append_tree(q, k, v, dev(c["cos"]), dev(c["sin"]), kc, vc, dev(c["table"]), dev(c["cu"]), dev(c["used"]),
                          dev(c["parent"]), interleaved=c["interleaved"], out=out, **kw)
    torch.cuda.synchronize()
    return out, kc, vc


def append_check(c, dt, got, in_place=False):
    out, kc, vc = got
    h, hk = c["h"], c["hk"]
    q, k, v = c["x"][:, :h], c["x"][:, h:h + hk], c["x"][:, h + hk:]
    pl = ref.places(c["cu"], c["used"], c["parent"], c["table"], q.shape[0], c["page"], c["pool"],
                    len(c["cos"]) if c["r"] else None)
    pos = np.array([p[1] for p in pl])
    q64, k64 = (paged.rotate(y, c["cos"][pos], c["sin"][pos], c["interleaved"]) for y in (q, k))
    want_q = q.astype(np.float64) if in_place else np.full(q.shape, 9.0)
    want_k = np.full(tuple(kc.shape), 9.0)
    want_v, ek = want_k.copy(), np.zeros(want_k.shape[:3] + (1,))
    for t, (seq, _, page, row) in enumerate(pl):
        if seq < 0:
            continue
        want_q[t] = q64[t]
        if page >= 0:
            want_k[page, row], want_v[page, row], ek[page, row] = k64[t], v[t], rotation_error(k[t])
    close(host(out), want_q, dt, rotation_error(q) if h else 0.0, "q")
    close(host(kc), want_k, dt, ek, "k")
    assert np.array_equal(host(vc), want_v.astype(np.float32))


@pytest.mark.parametrize("dt", sorted(T))
@pytest.mark.parametrize("case", sorted(APPEND))
def test_append(case, dt):
    c = append_case(case, dt)
    append_check(c, dt, append_run(c, dt))


@pytest.mark.parametrize("case", ["trees", "odd_d"])
def test_append_queries_in_place(case):
    c = append_case(case, "bfloat16")
    append_check(c, "bfloat16", append_run(c, "bfloat16", in_place=True), in_place=True)


def test_append_chain_is_the_plain_append():
    c = append_case("chain", "float16")
    x, h, hk = dev(c["x"], "float16"), c["h"], c["hk"]
    got = append_run(c, "float16")
    kc, vc = torch.full_like(got[1], 9.0), torch.full_like(got[2], 9.0)
    q = torch.full_like(got[0], 9.0)
    ops.paged_append(x[:, :h], x[:, h:h + hk], x[:, h + hk:], dev(c["cos"]), dev(c["sin"]), kc, vc, dev(c["table"]),
                     dev(c["cu"]), dev(c["used"]), out=q, sync=True)
    assert torch.equal(q, got[0]) and torch.equal(kc, got[1]) and torch.equal(vc, got[2])


def test_append_bad_places():
    """Pages outside the pool and the table, positions below 0 and past the tables of cos
    and sin, sequences outside the tokens: left out, the rest done."""
    for dt in ("bfloat16", "float32"):
        c = append_case("trees", dt)
        c["table"][0, 0], c["table"][2, 0] = -3, c["pool"]
        c["cos"], c["sin"] = c["cos"][:67], c["sin"][:67]  # the deeper nodes of sequence 0 lie past them
        append_check(c, dt, append_run(c, dt))
        c["used"][2] = 6                                   # base -3: roots at position -3, some below at 0 and past
        append_check(c, dt, append_run(c, dt))
        c["cu"][3] = c["x"].shape[0] + 1
        append_check(c, dt, append_run(c, dt))
        c["cu"][:] = [5, 2, -7, 1 << 30]
        append_check(c, dt, append_run(c, dt))


# ---------------------------------------------------------------- attention
ATTEND = {
    "one_key": dict(ql=[1], kl=[1], h=4, hk=4, d=128, page=64),
    "only_trees": dict(ql=[26, 7], kl=[26, 7], h=8, hk=2, d=128, page=16),
    "tile_edges": dict(ql=[3, 1, 2, 4], kl=[15, 32, 65, 129], h=8, hk=2, d=128, page=16),
    "rows32": dict(ql=[8, 3], kl=[700, 300], h=8, hk=2, d=128, page=16),
    "rows33": dict(ql=[11, 5], kl=[300, 40], h=3, hk=1, d=128, page=16),
    "rows64": dict(ql=[16, 13], kl=[500, 13], h=8, hk=2, d=64, page=32),
    "rows65": dict(ql=[65, 2], kl=[200, 70], h=2, hk=2, d=64, page=64),
    "rows128": dict(ql=[32, 9, 17], kl=[1000, 300, 64], h=8, hk=2, d=128, page=64),
    "rows129": dict(ql=[43, 30], kl=[400, 77], h=6, hk=2, d=128, page=64),
    "parts": dict(ql=[26, 1, 9], kl=[4000, 30, 1500], h=8, hk=2, d=128, page=64),
    "parts_d64": dict(ql=[13, 7], kl=[3051, 2300], h=8, hk=1, d=64, page=16),
    "parts_one": dict(ql=[1, 1, 1], kl=[4000, 1, 333], h=8, hk=2, d=128, page=64),
    "parts_blocks": dict(ql=[64, 50], kl=[2500, 1100], h=16, hk=2, d=128, page=64),
    "longest_parts": dict(ql=[5], kl=[16405], h=8, hk=1, d=128, page=64),
    "d256": dict(ql=[5, 2], kl=[600, 77], h=8, hk=2, d=256, page=32),
    "d256_blocks": dict(ql=[40, 9], kl=[1600, 77], h=8, hk=2, d=256, page=32),
    "chain": dict(ql=[70, 5], kl=[200, 5], h=4, hk=2, d=128, page=16, kinds=["chain"]),
    "forest": dict(ql=[64, 65, 7], kl=[64, 100, 30], h=4, hk=2, d=64, page=16, kinds=["forest"]),
    "star": dict(ql=[40, 64], kl=[50, 700], h=4, hk=2, d=128, page=64, kinds=["star"]),
    "large": dict(ql=[500, 1024], kl=[900, 1100], h=2, hk=1, d=64, page=64, kinds=["tree", "forest"]),
    "window": dict(ql=[26, 8], kl=[900, 80], h=8, hk=2, d=128, page=16, left=100),
    "window_parts": dict(ql=[26, 8], kl=[4000, 1980], h=8, hk=2, d=64, page=64, left=1900),
    "window_tree": dict(ql=[40, 30], kl=[300, 30], h=4, hk=2, d=128, page=16, left=2, kinds=["chain", "tree"]),
    "window_none": dict(ql=[9, 30], kl=[80, 31], h=4, hk=2, d=64, page=16, left=0),
    "fewer_keys_than_nodes": dict(ql=[8, 13], kl=[5, 1], h=2, hk=1, d=64, page=16),
    "no_keys_no_nodes": dict(ql=[3, 0, 2, 1], kl=[0, 40, 2, 500], h=4, hk=2, d=128, page=16),
    "page48": dict(ql=[11, 2], kl=[400, 100], h=4, hk=4, d=128, page=48),
    "page1": dict(ql=[11, 2], kl=[70, 9], h=4, hk=2, d=64, page=1),
    "page10": dict(ql=[7, 2], kl=[170, 9], h=4, hk=2, d=128, page=10),
    "odd_d": dict(ql=[12, 1], kl=[70, 300], h=4, hk=2, d=80, page=16),
    "d1": dict(ql=[6], kl=[70], h=2, hk=1, d=1, page=16),
    "many_parts": dict(ql=[1 + i % 5 for i in range(70)], kl=[540 + 97 * i % 1500 for i in range(70)], h=4, hk=1, d=64,
                       page=16),
    "part_edges": dict(ql=[2] * 24, kl=[514 + 61 * i for i in range(24)], h=4, hk=1, d=128, page=64),
    "part_edges_window": dict(ql=[3, 1] * 12, kl=[514 + 61 * i for i in range(24)], h=4, hk=1, d=64, page=64, left=700),
    "wide_parts": dict(ql=[60, 51, 64, 33], kl=[700, 900, 64, 1300], h=32, hk=8, d=128, page=64),
    "wide_parts_d64": dict(ql=[60, 51, 64, 33, 41], kl=[700, 900, 64, 1300, 41], h=32, hk=8, d=64, page=16),
    "d256_parts": dict(ql=[5, 2], kl=[2600, 1077], h=8, hk=2, d=256, page=32),
    "batch": dict(ql=[26 - i % 20 for i in range(40)], kl=[1100 - 25 * i for i in range(40)], h=8, hk=2, d=128, page=64),
}


def attend_case(name, dt, seed=0):
    c = dict(ATTEND[name]) if isinstance(name, str) else dict(name)
    rng = np.random.default_rng(seed)
    cu, used, table, pool = lists(c["ql"], c["kl"], c["page"], rng)
    rnd = paged.rounder(dt)
    k, v = (rng.standard_normal((pool, c["page"], c["hk"], c["d"])).astype(np.float32) for _ in range(2))
    k[..., 0] *= 3.0
    c.update(cu=cu, used=used, table=table, pool=pool, left=c.get("left", -1), parent=forest(c, rng),
             q=rnd(rng.standard_normal((sum(c["ql"]) + 3, c["h"], c["d"])).astype(np.float32) * 1.5), k=rnd(k), v=rnd(v),
             seqlen_q=c.get("seqlen_q", max(c["ql"])), seqlen_k=max(c["kl"]), scale=c.get("scale", 1 / math.sqrt(c["d"])))
    return c


def attend_args(c, dt):
    return (dev(c["q"], dt), dev(c["k"], dt), dev(c["v"], dt), dev(c["table"]), dev(c["cu"]), dev(c["used"]),
            dev(c["parent"]), c["seqlen_q"], c["seqlen_k"])


def attend_run(c, dt, args=None, **kw):
    args = attend_args(c, dt) if args is None else args
    o = torch.full(c["q"].shape, 9.0, dtype=T[dt], device="cuda")
    lse = torch.full((c["h"], c["q"].shape[0]), 9.0, device="cuda")
    ops.paged_attention_tree(*args, scale=c["scale"], window_left=c["left"], out=o, lse=lse, **kw)
    torch.cuda.synchronize()
    return o, lse


def attend_check(c, dt, o, lse):
    want, wl, rows, b = ref.attention(c["q"], c["k"], c["v"], c["cu"], c["used"], c["parent"], c["table"], c["scale"],
                                      c["left"], c["seqlen_q"])
    o, lse = host(o).astype(np.float64), host(lse).astype(np.float64)
    assert (o[~rows] == 9.0).all() and (lse[:, ~rows] == 9.0).all()
    half = torch.finfo(T[dt]).eps / 2
    e = U * c["d"] * b["qk"] + 6 * U / 2 * b["top"] + 2.0 ** -22
    bar = (2 * e + U * (b["keys"] + 64))[..., None] * b["pv"] + half * np.abs(want) + 2.0 ** -126
    if dt != "float32":
        bar += half * b["pv"] + torch.finfo(T[dt]).smallest_normal * torch.finfo(T[dt]).eps
        bar += 2.0 ** -25 * b["av"] if dt == "float16" else 0.0
    bad = ~(np.abs(o - want) <= bar)[rows]
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4], float(np.abs(o - want)[rows][bad].max()))
    none = np.isinf(wl)
    assert (lse[:, rows][none[:, rows]] == np.inf).all()
    fin = np.where(none, 0.0, wl)
    bad = ~(np.abs(lse - fin) <= e.T + 2.0 ** -20 * (1 + np.abs(fin) / 2))[:, rows] & ~none[:, rows]
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4])


@pytest.mark.parametrize("dt", sorted(T))
@pytest.mark.parametrize("case", sorted(ATTEND))
def test_attend(case, dt):
    c = attend_case(case, dt)
    attend_check(c, dt, *attend_run(c, dt))


# the last kernel of some of them (behind g950_attn_tree_<type>_): every form by name
FORMS = {"one_key": "d128_r2", "rows64": "d64_r2", "rows33": "d128_r2", "rows65": "d64_r4", "rows128": "d128_r4_merge4",
         "chain": "d128_r4", "large": "d64_r4_merge4", "d256": "d256_r2_merge16", "d256_blocks": "d256_r4_merge4",
         "longest_parts": "d128_r2_merge16", "parts_d64": "d64_r4_merge16", "wide_parts": "d128_r4_merge1",
         "wide_parts_d64": "d64_r4_merge1", "part_edges": "d128_r2_merge16", "many_parts": "d64_r2_merge4", "page48": "d128_r2",
         "page1": "general", "page10": "general", "odd_d": "general", "d1": "general"}


@pytest.mark.parametrize("case", sorted(FORMS))
def test_attend_forms(case):
    attend_run(attend_case(case, "float16"), "float16")
    assert rt.module().last_kernel == "g950_attn_tree_" + ("" if FORMS[case] == "general" else "f16_") + FORMS[case]


@pytest.mark.parametrize("floats", [0, 5000, 1 << 22])
def test_attend_any_workspace(floats):
    for case in ("parts", "parts_blocks", "window_parts"):
        c = attend_case(case, "bfloat16", seed=2)
        attend_check(c, "bfloat16", *attend_run(c, "bfloat16", workspace=torch.full((floats,), float("nan"), device="cuda")))


@pytest.mark.parametrize("dt", ["bfloat16", "float16", "float32"])
def test_attend_bad_lists(dt):
    """Pages outside the pool, a table too short, sequences outside the rows, lengths below the nodes."""
    c = attend_case("parts", dt)
    c["table"][0, 3], c["table"][0, 62], c["table"][2, 0] = -1, c["pool"], 1 << 30
    attend_check(c, dt, *attend_run(c, dt))
    c["table"] = np.ascontiguousarray(c["table"][:, :50])
    attend_check(c, dt, *attend_run(c, dt))
    c["used"][:] = [-(1 << 31), 1 << 20, -5]
    attend_check(c, dt, *attend_run(c, dt))
    c["cu"][:] = [0, 26, c["q"].shape[0] + 1, 4]
    attend_check(c, dt, *attend_run(c, dt))


@pytest.mark.parametrize("left", [-1, 40, 2 ** 31 - 1])
def test_attend_tables_that_end_before_the_tree(left):
    """The last key that the table holds and the tree's first in one tile: no node of the tree has a row."""
    for ql, kl, pages in (([5, 3], [59, 57], 3), ([5, 9], [1305, 1309], 81), ([26, 40], [80, 101], 4)):
        c = attend_case(dict(ql=ql, kl=kl, h=8, hk=2, d=128, page=16, left=left), "bfloat16")
        c["table"] = np.ascontiguousarray(c["table"][:, :pages])
        attend_check(c, "bfloat16", *attend_run(c, "bfloat16"))


def test_attend_the_widest_window():
    for case in ("fewer_keys_than_nodes", "parts_d64", "rows129"):
        c = dict(attend_case(case, "bfloat16"), left=2 ** 31 - 1)
        attend_check(c, "bfloat16", *attend_run(c, "bfloat16"))


@pytest.mark.parametrize("most", [0, 1, 20])
def test_attend_covers_seqlen_q_nodes(most):
    for case in ("parts", "rows129"):
        c = dict(attend_case(case, "bfloat16"), seqlen_q=most)
        attend_check(c, "bfloat16", *attend_run(c, "bfloat16"))


@pytest.mark.parametrize("dt", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("case", ["rows128", "parts_d64", "d256", "page10"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_unseen_keys_may_hold_anything(case, dt, bad):
    """NaN and infinities in the rows that no node sees (behind the sequences, unused pages), and in a
    node's own K and V: those that do not see it stay as they are."""
    c = attend_case(case, dt)
    hit, at = {}, set()
    for z in range(len(c["ql"])):
        base = c["kl"][z] - c["ql"][z]
        at |= {(c["table"][z, j // c["page"]], j % c["page"]) for j in range(c["kl"][z])}
        if c["ql"][z] > 3:
            hit[z] = 2
    clean = dict(c, k=c["k"].copy(), v=c["v"].copy())
    dirty = dict(c, k=c["k"].copy(), v=c["v"].copy())
    for pg in range(c["pool"]):
        for r in range(c["page"]):
            if (pg, r) not in at:
                dirty["k"][pg, r], dirty["v"][pg, r] = bad, bad
    a, b = attend_run(clean, dt), attend_run(dirty, dt)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    rows = np.zeros(c["q"].shape[0], bool)
    for z, x in hit.items():
        slot = c["kl"][z] - c["ql"][z] + x
        where = (c["table"][z, slot // c["page"]], slot % c["page"])
        dirty["v"][where], dirty["k"][where][..., :1] = bad, bad
        rows[[int(c["cu"][z]) + i for i in range(c["ql"][z]) if x in ref.way(c["parent"], int(c["cu"][z]), i)]] = True
    b = attend_run(dirty, dt)
    same = torch.from_numpy(~rows).cuda()
    assert torch.equal(a[0][same], b[0][same]) and torch.equal(a[1][:, same], b[1][:, same])
    assert rows.any() and not torch.isfinite(b[0][~same].float()).any(-1).all()


@pytest.mark.parametrize("bad", [float("inf"), float("-inf")])
@pytest.mark.parametrize("case", ["rows128", "parts_d64", "page10"])
def test_seen_infinities_come_through(case, bad):
    """An infinite value in V of a seen node: that infinity, in its dim alone."""
    c = attend_case(case, "bfloat16")
    z, x = 0, 0
    slot = c["kl"][z] - c["ql"][z] + x
    at = (c["table"][z, slot // c["page"]], slot % c["page"])
    a = attend_run(c, "bfloat16")
    c["v"][at][..., 5] = bad
    b = attend_run(c, "bfloat16")
    rows = torch.zeros(c["q"].shape[0], dtype=torch.bool, device="cuda")
    rows[[int(c["cu"][z]) + i for i in range(c["ql"][z]) if x in ref.way(c["parent"], int(c["cu"][z]), i)]] = True
    assert (b[0][rows][..., 5] == bad).all()
    a[0][rows, :, 5] = b[0][rows, :, 5]
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dt", ["bfloat16", "float32"])
def test_attend_strides(dt):
    """Head-major queries and outputs, a cache of head-major pages and one without 16-byte rows, in place."""
    for case in ("rows128", "parts"):
        c = attend_case(case, dt)
        q, k, v, *rest = attend_args(c, dt)
        hm = lambda x: x.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
        pad = lambda x: torch.nn.functional.pad(x, (0, 3))[..., :x.shape[-1]]  # noqa: E731
        qh = q.transpose(0, 1).contiguous().transpose(0, 1)
        for args in ((qh, hm(k), hm(v), *rest), (q, pad(k), pad(v), *rest), (pad(q), k, v, *rest)):
            attend_check(c, dt, *attend_run(c, dt, args))
        lse = torch.full((c["q"].shape[0], c["h"]), 9.0, device="cuda").t()
        ops.paged_attention_tree(q, k, v, *rest, scale=c["scale"], out=q, lse=lse, sync=True)
        _, _, rows, _ = ref.attention(c["q"], c["k"], c["v"], c["cu"], c["used"], c["parent"], c["table"], c["scale"], -1,
                                      c["seqlen_q"])
        o = q.clone()
        o[torch.from_numpy(~rows).cuda()] = 9.0
        attend_check(c, dt, o, lse)


def test_attend_a_chain_is_causal_attention():
    """A chain of nodes against the varlen kernel's paged causal attention, within both bars."""
    c = attend_case("chain", "bfloat16")
    o, lse = attend_run(c, "bfloat16")
    attend_check(c, "bfloat16", o, lse)
    p = [c["parent"][i] for i in range(70)]
    assert p == [i - 1 for i in range(70)]
    at = ref.seen(c["cu"], c["used"], c["parent"], c["table"], c["q"].shape[0], 16, c["pool"], -1, 70, 0)
    assert [len(x) for x in at] == [131 + i for i in range(70)]


# ------------------------------------------------------------- verification
VERIFY = {
    "one": dict(ql=[1], v=1000),
    "chain": dict(ql=[6, 3], v=1000, kinds=["chain"]),
    "trees": dict(ql=[26, 1, 9, 0, 13], v=1000),
    "star": dict(ql=[12, 30], v=500, kinds=["star"]),
    "v1": dict(ql=[4, 2], v=1),
    "v2": dict(ql=[9, 2], v=2),
    "v63": dict(ql=[26, 9], v=63),
    "odd": dict(ql=[26, 9], v=1025),
    "odd_large": dict(ql=[26], v=50257),
    "large": dict(ql=[9, 12], v=128000),
    "forest": dict(ql=[70, 130], v=300, kinds=["forest"]),
    "deep": dict(ql=[200, 64, 65], v=130, kinds=["tree", "chain", "star"]),
    "past_the_limit": dict(ql=[1100, 1024], v=40, kinds=["tree", "chain"]),
    "batch": dict(ql=[1 + i % 30 for i in range(300)], v=257),
}


def verify_case(name, drafts, dt, seed=0, sharp=2.0):
    c = dict(VERIFY[name])
    rng = np.random.default_rng(seed)
    t, v = sum(c["ql"]) + 2, c["v"]
    rnd = paged.rounder(dt)
    x = rng.standard_normal((t, v)) * sharp
    soft = lambda y: rnd((np.exp(y - y.max(-1, keepdims=True)) / np.exp(y - y.max(-1, keepdims=True)).sum(  # noqa: E731
        -1, keepdims=True)).astype(np.float32))
    c.update(target=soft(x), draft=soft(0.9 * x + 0.7 * rng.standard_normal((t, v))), parent=forest(c, rng)[:t],
             cu=np.cumsum([0] + c["ql"]).astype(np.int32), u=rng.random(t).astype(np.float32),
             last=rng.random(len(c["ql"])).astype(np.float32), tokens=rng.integers(0, v, t), distinct=drafts == "distinct")
    c["most"] = c.get("most", 12)
    for z, n in enumerate(c["ql"]):
        b0 = int(c["cu"][z])
        for cur in range(min(n, 200)):
            kids = [i for i in range(1, n) if c["parent"][b0 + i] == cur]
            w = (c["draft"] if drafts != "chosen" else c["target"])[b0 + cur].astype(np.float64) + 1e-30
            w = w / w.sum()
            put = len(kids) if drafts == "drawn" else min(len(kids), v)
            c["tokens"][[b0 + i for i in kids[:put]]] = rng.choice(v, put, replace=drafts == "drawn", p=w)
    if drafts == "chosen":
        c["draft"] = None
    return c


def verify_run(c, dt, token=torch.int64, pad=0, **kw):
    def rows(x):
        if x is None:
            return None
        x = dev(x, dt)
        return torch.nn.functional.pad(x, (0, pad))[:, :x.shape[1]] if pad else x
    got = ops.verify_tree(rows(c["target"]), rows(c["draft"]), dev(c["tokens"]).to(token), dev(c["parent"]), dev(c["u"]),
                          dev(c["last"]), dev(c["cu"]), c["most"], distinct=c["distinct"], sync=True, **kw)
    return [x.cpu().numpy() for x in got]


def verify_check(c, got):
    want = ref.verify(c["target"], c["draft"], c["tokens"], c["parent"], c["u"], c["last"], c["cu"], c["most"],
                      c["distinct"])
    for name, g, w in zip(("path", "count", "next"), got, want):
        assert np.array_equal(g, w), (name, np.argwhere(g != w)[:5], g[g != w][:5], w[g != w][:5])


@pytest.mark.parametrize("dt", sorted(T))
@pytest.mark.parametrize("drafts", ["drawn", "distinct", "chosen"])
@pytest.mark.parametrize("case", sorted(VERIFY))
def test_verify(case, drafts, dt):
    c = verify_case(case, drafts, dt)
    verify_check(c, verify_run(c, dt))


@pytest.mark.parametrize("drafts", ["drawn", "distinct", "chosen"])
def test_verify_seeds(drafts):
    """Paths of all lengths: many numbers over the same trees, peaked and flat rows."""
    lengths = set()
    for seed in range(12):
        c = verify_case("trees", drafts, "float32", seed=seed, sharp=[1.0, 3.0, 6.0][seed % 3])
        got = verify_run(c, "float32", token=torch.int32)
        verify_check(c, got)
        lengths |= set(got[1].tolist())
    assert lengths >= {0, 1, 2, 3}


@pytest.mark.parametrize("drafts", ["drawn", "distinct", "chosen"])
def test_verify_any_workspace(drafts):
    """One workgroup a sequence, several and as many as are wanted: the same answers."""
    for case in ("large", "odd_large"):
        c = verify_case(case, drafts, "bfloat16", seed=1)
        t, b = c["target"].shape[0], len(c["ql"])
        for parts in (0, 1, 2, 7, 64):
            ws = torch.full((t * 4 + b * 64 * parts,), float("nan"), device="cuda")
            verify_check(c, verify_run(c, "bfloat16", workspace=ws))


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
def test_verify_many_refusals(dt):
    """A root with 90 children, nearly all of them refused: more sums than the workgroups tell each
    other, the rest each adds up by itself."""
    VERIFY["refused"] = dict(ql=[91, 60], v=9000, kinds=["star"])
    c = verify_case("refused", "drawn", dt, seed=2)
    c["u"][:] = 1 - 2.0 ** -24
    for ws in (None, torch.empty(0, device="cuda")):
        got = verify_run(c, dt, workspace=ws)
        verify_check(c, got)
    c["tokens"][1:80] = int(c["target"][0].argmin())
    verify_check(c, verify_run(c, dt))


@pytest.mark.parametrize("drafts", ["drawn", "chosen"])
def test_verify_wide_levels(drafts):
    """Each level's children spread over several 64-node windows, all refused but the last one."""
    VERIFY["wide"] = dict(ql=[600, 1], v=3001)
    for seed in range(3):
        c = verify_case("wide", drafts, "float32", seed=seed)
        c["parent"][1:600] = [-1 if i < 1 else 199 * ((i - 1) // 199) for i in range(1, 600)]
        c["tokens"][:600] = np.random.default_rng(seed).permutation(3001)[:600]
        c["u"][:] = 1 - 2.0 ** -24
        c["u"][[199, 398, 597]] = 0.0
        for ws in (None, torch.empty(0, device="cuda")):
            got = verify_run(c, "float32", workspace=ws)
            verify_check(c, got)
            if drafts == "chosen":
                assert got[0][0, :4].tolist() == [0, 199, 398, 597]


def test_verify_unbounded_drafts():
    """A draft's value that is infinite takes its column from what is left, but not from p, which is
    taken where nothing is left."""
    VERIFY["two"] = dict(ql=[2], v=9000)
    c = verify_case("two", "drawn", "float32")
    c["parent"][:2], c["tokens"][1], c["u"][1], c["last"][0] = [-1, 0], 3, 1 - 2.0 ** -24, 0.5
    c["target"][0] = 0.125 / 8999
    c["target"][0, 5000] = 0.875
    c["draft"][0] = c["target"][0] * 2
    c["draft"][0, 5000] = np.inf
    for ws in (None, torch.empty(0, device="cuda")):
        path, count, nxt = verify_run(c, "float32", workspace=ws)
        assert count.tolist() == [1] and nxt.tolist() == [5000] and path[0, 0] == 0


@pytest.mark.parametrize("most", [1, 2, 3])
def test_verify_full_paths(most):
    for drafts in ("drawn", "chosen"):
        c = dict(verify_case("chain", drafts, "float32"), most=most)
        c["u"][:] = 0.0
        got = verify_run(c, "float32")
        verify_check(c, got)
        assert (got[1] == most).all()


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
def test_verify_special_rows(dt):
    """Numbers at their ends, tokens outside the vocabulary and repeated, rows of one token, of
    zeros, with NaN and below zero; equal rows."""
    for drafts in ("drawn", "distinct", "chosen"):
        c = verify_case("trees", drafts, dt, seed=3)
        c["last"][:] = [0.0, 1 - 2.0 ** -24, 0.5, 0.25, 1 - 2.0 ** -24]
        c["u"][::3] = 0.0
        c["u"][1::3] = 1 - 2.0 ** -24
        c["target"][:, 500:] = 0.0      # nothing behind column 500
        verify_check(c, verify_run(c, dt))
        c["tokens"][::4], c["tokens"][2::16] = -1, 1000
        c["tokens"][3::8] = 1 << 40
        verify_check(c, verify_run(c, dt))
        if drafts != "distinct":
            c["tokens"][1:20] = 7       # repeated
            verify_check(c, verify_run(c, dt))
        c["target"][5:9, :] = 0.0
        c["target"][5:9, 499] = 1.0
        c["target"][0, 20:30] = -0.5
        c["target"][1, 20:30] = np.nan
        verify_check(c, verify_run(c, dt))
        c = verify_case("trees", drafts, dt, seed=4)
        if drafts != "chosen":
            c["draft"] = c["target"].copy()   # nothing is refused but what the draft could not draw
            c["u"][:] = 1 - 2.0 ** -24
            verify_check(c, verify_run(c, dt))
        c["target"][:] = 0.0            # nothing at all: token 0
        got = verify_run(c, dt)
        verify_check(c, got)
        assert set(got[2].tolist()) == {0, -1}


@pytest.mark.parametrize("pad", [1, 8])
def test_verify_strides(pad):
    """Rows that are not multiples of 16 bytes apart."""
    for dt in sorted(T):
        for case in ("trees", "odd", "odd_large"):
            c = verify_case(case, "drawn", dt, seed=6)
            verify_check(c, verify_run(c, dt, pad=pad))


def test_verify_bad_lists():
    c = verify_case("trees", "drawn", "float32")
    for cu in ([0, 26, 27, 1 << 30, 36, 49], [5, 2, -7, 1 << 30, 4, 60]):
        c["cu"][:] = cu
        verify_check(c, verify_run(c, "float32"))


# ------------------------------------------------------ the accepted path's rows
KEEP = {
    "one": dict(ql=[1], kl=[1], hk=8, d=128, page=16),
    "trees": dict(ql=[26, 1, 9, 0, 40], kl=[90, 40, 9, 3, 100], hk=2, d=128, page=64),
    "layers": dict(ql=[26, 9], kl=[90, 9], hk=4, d=64, page=16, layers=5),
    "odd_d": dict(ql=[14, 13], kl=[14, 31], hk=3, d=77, page=7),
    "d2": dict(ql=[14, 13], kl=[14, 31], hk=1, d=2, page=16),
    "many_heads": dict(ql=[20], kl=[31], hk=40, d=256, page=16),
    "page1": dict(ql=[20, 5], kl=[31, 5], hk=2, d=64, page=1),
    "long": dict(ql=[300], kl=[400], hk=2, d=32, page=16, long=True),
    "batch": dict(ql=[17] * 90, kl=[20 + i for i in range(90)], hk=2, d=64, page=16),
}


def keep_case(name, dt, seed=0):
    c = dict(KEEP[name])
    rng = np.random.default_rng(seed)
    cu, used, table, pool = lists(c["ql"], c["kl"], c["page"], rng)
    most = max(c["ql"]) + 2
    path, count = np.full((len(used), most), -1, np.int32), np.zeros(len(used), np.int32)
    for z, n in enumerate(c["ql"]):
        k = n * 2 // 3 if c.get("long") else int(rng.integers(0, min(n, 9) + 1))
        path[z, :k], count[z] = np.sort(rng.permutation(n)[:k]), k
    shape = (pool, c["page"], c["hk"], c["d"])
    shape = (c["layers"],) + shape if "layers" in c else shape
    c.update(cu=cu, used=used, table=table, pool=pool, path=path, count=count,
             k=paged.rounder(dt)(rng.standard_normal(shape).astype(np.float32)),
             v=paged.rounder(dt)(rng.standard_normal(shape).astype(np.float32)))
    return c


def keep_check(c, dt, make=lambda x: x):
    k, v = make(dev(c["k"], dt)), make(dev(c["v"], dt))
    used = ops.paged_keep_path(k, v, dev(c["table"]), dev(c["cu"]), dev(c["used"]), dev(c["path"]), dev(c["count"]), sync=True)
    for got, x in ((k, c["k"]), (v, c["v"])):
        want, left = ref.keep(x, c["cu"], c["used"], c["table"], c["path"], c["count"])
        assert np.array_equal(host(got), want)
    assert np.array_equal(used.cpu().numpy(), left)


@pytest.mark.parametrize("dt", sorted(T))
@pytest.mark.parametrize("case", sorted(KEEP))
def test_keep(case, dt):
    keep_check(keep_case(case, dt), dt)


def test_keep_any_path():
    """Paths that do not increase, entries outside the tree, counts past both, pages that are not there."""
    for seed in range(4):
        c = keep_case("trees", "bfloat16", seed)
        rng = np.random.default_rng(seed)
        c["path"] = rng.integers(-3, 45, c["path"].shape).astype(np.int32)
        c["count"] = np.array([100, 1, -4, 3, 42], np.int32)
        keep_check(c, "bfloat16")
        c["table"][0, 1], c["table"][4, 1] = -1, c["pool"]
        c["used"][1:3] = [0, -20]
        keep_check(c, "bfloat16")
        c["table"] = np.ascontiguousarray(c["table"][:, :1])
        keep_check(c, "bfloat16")
        c["cu"][2:4] = [1, 1 << 30]
        keep_check(c, "bfloat16")


def test_keep_without_layers():
    """Caches of no layers, and of no pages: the lengths are written."""
    c = keep_case("trees", "bfloat16")
    for shape in ((0, 4, 64, 2, 128), (0, 64, 2, 128)):
        k = torch.zeros(shape, dtype=torch.bfloat16, device="cuda")
        used = ops.paged_keep_path(k, k.clone(), dev(c["table"]), dev(c["cu"]), dev(c["used"]), dev(c["path"]),
                                   dev(c["count"]), sync=True)
        assert used.cpu().tolist() == (c["used"] - np.diff(c["cu"]) + c["count"]).tolist()


def test_keep_strides():
    for case, dt in (("trees", "bfloat16"), ("layers", "float32"), ("odd_d", "float16")):
        c = keep_case(case, dt)
        keep_check(c, dt, lambda x: x.transpose(-2, -3).contiguous().transpose(-2, -3))
        keep_check(c, dt, lambda x: torch.nn.functional.pad(x, (0, 3))[..., :x.shape[-1]])


# ------------------------------------------------------------ all of a step
def test_steps_of_drafted_trees_are_ordinary_decoding():
    """A one-layer model decodes by drafted trees: append, attention, softmax, verification,
    move.  Its cache, lengths and next outputs are those of the accepted tokens appended one after the other."""
    rng = np.random.default_rng(0)
    g = torch.Generator(device="cuda").manual_seed(0)
    h, hk, d, vocab, page, b, n = 8, 2, 128, 320, 16, 3, 14
    dt = torch.bfloat16
    emb = torch.randn((vocab, (h + 2 * hk) * d), generator=g, device="cuda").to(dt)
    head = torch.randn((h * d, vocab), generator=g, device="cuda") / 12
    cos, sin = (dev(x) for x in rope(200, d, rng))
    table = dev(rng.permutation(b * 12).reshape(b, 12).astype(np.int32))
    caches = [torch.zeros((b * 12, page, hk, d), dtype=dt, device="cuda") for _ in range(4)]
    split = lambda t: emb[t].view(-1, h + 2 * hk, d).split([h, hk, hk], 1)  # noqa: E731
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    # prompts of different lengths into both caches
    lens = [5, 31, 17]
    cu, used = ints(np.cumsum([0] + lens)), ints(lens)
    prompt = torch.randint(0, vocab, (sum(lens),), generator=g, device="cuda")
    q, k, v = split(prompt)
    for i in (0, 2):
        ops.paged_append(q, k, v, cos, sin, caches[i], caches[i + 1], table, cu, used)
    root = torch.randint(0, vocab, (b,), generator=g, device="cuda")
    cu = ints([0, n, 2 * n, 3 * n])
    accepted = 0
    for step in range(6):
        parent = np.concatenate([tree_of("tree", n, rng) for _ in range(b)]).astype(np.int32)
        tokens = torch.randint(0, vocab, (b, n), generator=g, device="cuda")
        tokens[:, 0] = root
        tokens = tokens.view(-1)
        now = used + n
        q, k, v = split(tokens)
        qr = ops.paged_append_tree(q, k, v, cos, sin, caches[0], caches[1], table, cu, now, dev(parent))
        o, _ = ops.paged_attention_tree(qr, caches[0], caches[1], table, cu, now, dev(parent), n, 200)
        probs = ops.softmax((o.view(-1, h * d).float() @ head))
        u = torch.rand(b * n, generator=g, device="cuda") * 0.004  # (drafts at random: refused otherwise)
        last = torch.rand(b, generator=g, device="cuda")
        path, count, nxt = ops.verify_tree(probs, None, tokens, dev(parent), u, last, cu, n)
        used = ops.paged_keep_path(caches[0], caches[1], table, cu, now, path, count)
        # the accepted tokens, appended as a chain behind the same keys
        kept = [tokens.view(b, n)[z, path[z, :count[z]].long()] for z in range(b)]
        c2 = ints(np.cumsum([0] + [len(x) for x in kept]))
        q2, k2, v2 = split(torch.cat(kept))
        qo = ops.paged_append(q2, k2, v2, cos, sin, caches[2], caches[3], table, c2, used)
        chain = ints([i - 1 for x in kept for i in range(len(x))])
        o2, lse2 = ops.paged_attention_tree(qo, caches[2], caches[3], table, c2, used, chain, n, 200)
        for z in range(b):
            assert int(used[z]) == int(now[z]) - n + int(count[z])
            j = torch.arange(int(used[z]), device="cuda")
            at = table[z, j // page].long()
            for i in range(2):
                assert torch.equal(caches[i][at, j % page], caches[i + 2][at, j % page]), (step, z)
            mine, theirs = (x.float() for x in (o.view(b, n, h, d)[z, path[z, :count[z]].long()], o2[c2[z]:c2[z + 1]]))
            # the same keys through other tiles: each within its bar of the same sums, 4 h max |V| at most
            assert (mine - theirs).abs().max() <= 4 * 2.0 ** -8 * float(caches[1].abs().max())
        accepted += int(count.sum()) - b
        root = nxt
    assert accepted > 0


# ------------------------------------------------- streams, graphs, devices
def test_streams_threads_and_graphs():
    """Calls on streams of their own from several threads, and captured graphs replayed in turn,
    give the eager call's bits."""
    c, w = attend_case("parts", "bfloat16"), verify_case("trees", "drawn", "float32")
    args = attend_args(c, "bfloat16")
    vargs = (dev(w["target"]), dev(w["draft"]), dev(w["tokens"]), dev(w["parent"]), dev(w["u"]), dev(w["last"]), dev(w["cu"]),
             w["most"])
    n = sum(c["ql"])  # (rows behind them are left as they are: whatever their memory held)

    def step(**kw):
        o, lse = ops.paged_attention_tree(*args, scale=c["scale"], **kw)
        return (o[:n], lse[:, :n]) + ops.verify_tree(*vargs, **kw)
    want = step()
    torch.cuda.synchronize()
    errors = []

    def work(i):
        try:
            s = own_stream(i)
            for _ in range(8):
                got = step(stream=s)
                s.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(got, want))
        except Exception as e:  # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors, errors
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = step()
        graphs.append((g, got))
    for _ in range(3):
        for g, got in graphs:
            for x in got:
                x.zero_()
            g.replay()
            eager = step()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            assert torch.equal(eager[0], want[0])


def test_captured_step():
    """Append, verification and move in one graph, replayed on new inputs in place."""
    c, k = append_case("trees", "bfloat16"), keep_case("trees", "bfloat16")
    x, h, hk = dev(c["x"], "bfloat16"), c["h"], c["hk"]
    cos, sin, table, cu, used, parent = (dev(c[n]) for n in ("cos", "sin", "table", "cu", "used", "parent"))
    kc = torch.full((c["pool"], c["page"], hk, c["d"]), 9.0, dtype=torch.bfloat16, device="cuda")
    vc = kc.clone()
    kk, kv = dev(k["k"], "bfloat16"), dev(k["v"], "bfloat16")
    lists_ = [dev(k[n]) for n in ("table", "cu", "used", "path", "count")]
    ops.paged_append_tree(x[:, :h], x[:, h:h + hk], x[:, h + hk:], cos, sin, kc.clone(), vc.clone(), table, cu, used, parent)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q = ops.paged_append_tree(x[:, :h], x[:, h:h + hk], x[:, h + hk:], cos, sin, kc, vc, table, cu, used, parent)
        left = ops.paged_keep_path(kk, kv, *lists_)
    for seed in range(3):
        c2, k2 = append_case("trees", "bfloat16", seed + 5), keep_case("trees", "bfloat16", seed + 5)
        for t, s in ((x, c2["x"]), (kk, k2["k"]), (kv, k2["v"])):
            t.copy_(dev(s, "bfloat16"))
        for t, s in zip((table, parent, *lists_), (c2["table"], c2["parent"], *(k2[n] for n in (
                "table", "cu", "used", "path", "count")))):
            t.copy_(dev(s))
        for t in (kc, vc, q):
            t.fill_(9.0)
        g.replay()
        torch.cuda.synchronize()
        for got, y in ((kk, k2["k"]), (kv, k2["v"])):
            want, used2 = ref.keep(y, k2["cu"], k2["used"], k2["table"], k2["path"], k2["count"])
            assert np.array_equal(host(got), want)
        assert np.array_equal(left.cpu().numpy(), used2)
        append_check(c2, "bfloat16", (q, kc, vc))


def test_outputs_keep_to_their_streams():
    """Tensors on other devices or the host are refused, before anything runs."""
    c = attend_case("rows32", "bfloat16")
    args = list(attend_args(c, "bfloat16"))
    for i in (0, 1, 3, 6):
        bad = list(args)
        bad[i] = bad[i].cpu()
        with pytest.raises(rt.G950Error):
            ops.paged_attention_tree(*bad, out=torch.empty_like(args[0]), lse=torch.empty((8, args[0].shape[0]), device="cuda"),
                                     workspace=torch.empty(0, device="cuda"))


def test_offsets_past_32_bits():
    """Pages and rows more than 2^31 elements in: the bits of the same calls on small tensors."""
    dt, page, hk, d, far = "bfloat16", 64, 8, 128, 40000
    c = attend_case(dict(ql=[26, 9], kl=[1500, 700], h=32, hk=hk, d=d, page=page), dt)
    x = dev(np.random.default_rng(1).standard_normal((c["q"].shape[0], 32 + 2 * hk, d)).astype(np.float32), dt)
    cos, sin = (dev(y) for y in rope(1500, d, np.random.default_rng(2)))
    k = keep_case("trees", dt)
    path, count = dev(k["path"][:2]), dev(k["count"][:2])
    path[0, :3], count[0] = torch.tensor([0, 5, 9], dtype=torch.int32, device="cuda"), 3
    path[1, :2], count[1] = torch.tensor([0, 8], dtype=torch.int32, device="cuda"), 2

    def run(kc, vc, table):
        q = ops.paged_append_tree(x[:, :32], x[:, 32:32 + hk], x[:, 32 + hk:], cos, sin, kc, vc, table, dev(c["cu"]),
                                  dev(c["used"]), dev(c["parent"]))
        o, lse = ops.paged_attention_tree(q, kc, vc, table, dev(c["cu"]), dev(c["used"]), dev(c["parent"]), 26, 1500)
        left = ops.paged_keep_path(kc, vc, table, dev(c["cu"]), dev(c["used"]), path, count)
        return q[:35], o[:35], lse[:, :35], left
    small = [dev(c[n], dt) for n in ("k", "v")]
    large = [torch.zeros((far + c["pool"], page, hk, d), dtype=T[dt], device="cuda") for _ in range(2)]
    for a, b in zip(large, small):
        a[far:] = b
    table = dev(c["table"])
    want, got = run(*small, table), run(*large, table + far)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    for a, b in zip(large, small):
        assert torch.equal(a[far:], b) and not a[:far].any()
    del large
    v, rows = 128000, 20000
    w = dict(verify_case("large", "drawn", dt))
    n = w["target"].shape[0]
    want = verify_run(w, dt)
    p, q = (torch.zeros((rows + n, v), dtype=T[dt], device="cuda") for _ in range(2))
    p[rows:], q[rows:] = dev(w["target"], dt), dev(w["draft"], dt)
    pad = lambda y: torch.cat([torch.zeros(rows, dtype=y.dtype, device="cuda"), y])  # noqa: E731
    for ws in (None, torch.empty(0, device="cuda")):
        got = ops.verify_tree(p, q, pad(dev(w["tokens"])), pad(dev(w["parent"])), pad(dev(w["u"])), dev(w["last"]),
                              dev(w["cu"]) + rows, w["most"], workspace=ws, sync=True)
        for a, b in zip(got, want):
            assert np.array_equal(a.cpu().numpy(), b)


@pytest.mark.parametrize("dt", ["bfloat16", "float32"])
def test_empty_batches(dt):
    """No sequences, no tokens, neither: nothing is written, and lengths and lists come out as they should."""
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    kc = torch.full((4, 16, 2, 64), 9.0, dtype=T[dt], device="cuda")
    vc = kc.clone()
    cos = sin = torch.ones((40, 32), device="cuda")
    for b, t in ((0, 3), (2, 0), (0, 0), (2, 3)):
        cu, used, parent = ints(*[0] * (b + 1)), ints(*[20] * b), ints(*[-1] * t)
        table = torch.zeros((b, 4), dtype=torch.int32, device="cuda")
        q, k, v = (torch.ones((t, n, 64), dtype=T[dt], device="cuda") for n in (4, 2, 2))
        out = torch.full_like(q, 9.0)
        ops.paged_append_tree(q, k, v, cos, sin, kc, vc, table, cu, used, parent, out=out)
        o, lse = torch.full_like(q, 9.0), torch.full((4, t), 9.0, device="cuda")
        ops.paged_attention_tree(q, kc, vc, table, cu, used, parent, 3, 800, out=o, lse=lse)
        p = torch.full((t, 7), 1 / 7, dtype=T[dt], device="cuda")
        path, count, nxt = ops.verify_tree(p, p, torch.zeros(t, dtype=torch.int64, device="cuda"), parent,
                                           torch.zeros(t, device="cuda"), torch.zeros(b, device="cuda"), cu, 5)
        left = ops.paged_keep_path(kc, vc, table, cu, used, path, count, sync=True)
        assert all((x == 9.0).all() for x in (kc, vc, out, o, lse))
        assert path.tolist() == [[-1] * 5] * b and count.tolist() == [0] * b and nxt.tolist() == [-1] * b
        assert left.tolist() == [20] * b


@pytest.mark.parametrize("drafts", ["drawn", "chosen"])
def test_verification_by_several_workgroups_at_once(drafts):
    """Calls of many parts on streams of their own from several threads, beside two captured graphs
    replayed in turn on new numbers: each the answers of its own inputs."""
    cases = [verify_case("large", drafts, "float32", seed=s) for s in range(3)]
    wants = [verify_run(c, "float32") for c in cases]
    for c, w in zip(cases, wants):
        verify_check(c, w)
    names = ("target", "draft", "tokens", "parent", "u", "last", "cu")
    inputs = [[None if c[n] is None else dev(c[n]) for n in names] for c in cases]
    most = cases[0]["most"]
    same = lambda got, want: all(np.array_equal(x.cpu().numpy(), y) for x, y in zip(got, want))  # noqa: E731
    slots = [[None if x is None else x.clone() for x in inputs[0]] for _ in range(2)]
    graphs = []
    for slot in slots:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = ops.verify_tree(*slot, most)
        graphs.append((g, got, slot))
    assert rt.module().last_kernel == "g950_verify_tree_f32_parts"
    errors = []

    def work(i):
        try:
            s = own_stream(i)
            for k in range(6):
                got = ops.verify_tree(*inputs[(i + k) % 3], most, stream=s)
                s.synchronize()
                assert same(got, wants[(i + k) % 3])
        except Exception as e:  # noqa: BLE001
            errors.append(e)
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    [t.start() for t in threads]
    for k in range(6):
        for n, (g, got, slot) in enumerate(graphs):
            for x, y in zip(slot, inputs[(k + n) % 3]):
                if x is not None:
                    x.copy_(y)
            g.replay()
        torch.cuda.current_stream().synchronize()
        for n, (g, got, slot) in enumerate(graphs):
            assert same(got, wants[(k + n) % 3])
    [t.join() for t in threads]
    assert not errors, errors
