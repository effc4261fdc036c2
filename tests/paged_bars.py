"""4-bit paged attention in float64 with the error that each output may have.

Bars, from the kernels' arithmetic (u = 2^-24, half a step of fp32; U = 2^-23, a whole
step, for the sums inside the matrix cores, whose rounding is not documented):

Score of a key with scale s and offset o: scale (s x + o Q), x = sum q c with c in -8 .. 7,
Q = sum q.  Q1 = sum |q|, Qm = the larger of the sums of the positive and of the
negative q (bounds every partial sum of q, in any order).
  * Q is summed in fp32: d / 8 + 3 additions on each element's way: (d / 8 + 3) u Q1 = eq.
  * x = -B Q + sum q (B + c), B = 136 in bfloat16 (codes biased by 128, 8 of them their
    own), 72 in float16: the first term has B (eq + u |Q|), the d additions of exact products
    one step each of a partial sum, which is at most B Qm + 8 Q1: U d (B Qm + 8 Q1).
  * s x + o Q: s, o and scale rounded into log2 units, a product, a sum: 6 u of each term,
    and o eq; the exponent's subtraction and exp2: 2 u of the score, 2^-22.
LSE is off by at most the largest error e of a score, and by 2^-20 (1 + |LSE| / 2) for its sum and log.

O = sum p V: p's relative errors e move it by e sum p |V - O|, p s rounds to bfloat16 (2^-8; a
second term in float16 models leaves 2^-16 of it) before it meets c: 2^-8 sum p s |c|; a wave's
sums of m keys, codes biased by 136, and the same once more for the bias: U m 2 (136 + 8) sum p s
(twice the additions with two terms); the offsets' and the denominator's sums u (m + 64)
of sum p |o| and |O|.  O rounds to its type once.
"""
import math

import numpy as np

from compiler_amd import runtime as rt
from oracle import paged as ref
from test_gpu_paged_int4 import attend_case

U = 2.0 ** -23
HALF = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"bfloat16": 2.0 ** -133, "float16": 2.0 ** -24}

# beside the cases of test_gpu_paged_int4: several blocks of query rows cut into several
# parts, windows over parts, sequences of one part beside long ones
MORE = {
    "blocks_parts": dict(ql=[40, 9], kl=[3000, 1200], h=8, hk=2, d=128, page=64),
    "blocks_parts_d64": dict(ql=[40, 9], kl=[3000, 1200], h=8, hk=2, d=64, page=16),
    "blocks_parts_d256": dict(ql=[21, 9], kl=[2200, 1200], h=8, hk=2, d=256, page=32),
    "blocks_parts_window": dict(ql=[40, 9, 3], kl=[3000, 1200, 70], h=8, hk=2, d=128, page=64, window=(700, 0)),
    "blocks_parts_window_d64": dict(ql=[50, 5], kl=[2500, 1100], h=6, hk=2, d=64, page=48, causal=False, window=(900, 11)),
    "parts_window": dict(ql=[1, 2, 1], kl=[4000, 1100, 90], h=8, hk=2, d=128, page=64, window=(1500, 0)),
    "parts_window_d64": dict(ql=[1, 2, 1], kl=[4000, 1100, 90], h=8, hk=2, d=64, page=16, window=(1500, 0)),
    "parts_window_d256": dict(ql=[2, 1], kl=[2000, 90], h=4, hk=2, d=256, page=16, causal=False, window=(1111, 5)),
    "short_beside_long": dict(ql=[3, 1, 2], kl=[4000, 30, 1500], h=4, hk=1, d=128, page=64),
    "group3_parts": dict(ql=[35, 2], kl=[2500, 400], h=3, hk=1, d=128, page=16),
    "noncausal_parts": dict(ql=[30, 4], kl=[2100, 1030], h=4, hk=2, d=64, page=64, causal=False),
    "longest_parts": dict(ql=[1], kl=[16400], h=8, hk=1, d=128, page=64),
    "wide_past_1024": dict(ql=[1] * 33, kl=[1300 - 40 * i for i in range(33)], h=16, hk=8, d=128, page=64),
}

# the last kernel of each case (after g950_attn_int4_<type>_d<dim>; "": the general one)
FORMS = {
    "one_key": "_r1", "tile_edges": "_r1", "round_edges": "_r1", "ranges": "_r1_merge", "ranges_d64": "_r1_merge",
    "d256": "_r1", "rows32": "_r2", "rows17": "_r2", "rows33": "_r2", "chunk": "_r2", "chunk_d64": "_r2", "group3": "_r1",
    "noncausal": "_r2", "local": "_r1w", "local_both": "_r2", "fewer_keys_than_queries": "_r1", "no_keys_no_queries": "_r1",
    "page48": "_r1", "page1": "", "page10": "", "wide": "_r1w", "wide_d64": "_r1w", "wide_few": "_r1w",
    "wide_few_d64": "_r1w", "odd_d": "", "d2": "",
    "blocks_parts": "_r2_merge", "blocks_parts_d64": "_r2_merge", "blocks_parts_d256": "_r1_merge",
    "blocks_parts_window": "_r2_merge", "blocks_parts_window_d64": "_r2_merge", "parts_window": "_r1_merge",
    "parts_window_d64": "_r1_merge", "parts_window_d256": "_r1_merge", "short_beside_long": "_r1_merge",
    "group3_parts": "_r2_merge", "noncausal_parts": "_r2_merge", "longest_parts": "_r1_merge", "wide_past_1024": "_r1w",
}


def aim(c, dt, strength=4.0):
    """Each query row (token, head) along one key of its sequence, which takes nearly all of its
    softmax: the first and the last key that it sees, the keys beside those
    that it does not see, a key of the second page, and others spread over all it sees."""
    r = 0
    for b, used in enumerate(c["used"]):
        b0, b1 = int(c["cu"][b]), int(c["cu"][b + 1])
        for i in range(b1 - b0):
            p0 = i + int(used) - (b1 - b0)
            right = 0 if c["causal"] else c["window"][1]
            first = max(0, p0 - c["window"][0]) if c["window"][0] >= 0 else 0
            last = min(int(used) - 1, p0 + right) if right >= 0 else int(used) - 1
            for hh in range(c["h"]):
                spread = first + r * 97 % max(last - first + 1, 1)
                j = [first, last, first - 1, last + 1, c["page"], spread, spread, spread][r % 8]
                j = min(max(j, 0), int(used) - 1)
                r += 1
                if j < 0:
                    continue
                at, kv = c["table"][b, j // c["page"]], hh // (c["h"] // c["hk"])
                key = ref.values(c["kc"][at, j % c["page"], kv], c["ks"][at, j % c["page"], kv])
                c["q"][b0 + i, hh] = ref.rounder(dt)((strength * key).astype(np.float32))
    return c


def case(name, dt, seed=0, aimed=False):
    c = attend_case(MORE[name] if name in MORE else name, dt, seed)
    return aim(c, dt) if aimed else c


def kernel_of(name, c, dt):
    t = "bf16" if dt == "bfloat16" else "f16"
    return f"g950_attn_int4_{t}_d{c['d']}{FORMS[name]}" if FORMS[name] else "g950_attn_int4_general"


def bf16_step(x):
    """Rounded to bfloat16, in float64."""
    return ref.bf16_round(x.astype(np.float32)).astype(np.float64)


def attend(c, dt, bars=True, parts=None, later=0, scale=1.0, codes=0, offsets=1.0, scales=1.0, without=None, once=False, zero=False):
    """o, lse [h, t], rows written and, with ``bars``, the bars of o and lse, for a call of
    ``parts`` at most (default: as many as its sizes ask for).  The other arguments compute something else on purpose: the causal (or window's) end
    ``later``, the softmax scale times ``scale``, V's ``codes`` off, its ``offsets`` and
    ``scales`` times these, keys ``without`` a column of the page table, p s rounded to bfloat16
    ``once``, V ``zero``."""
    t, h, d = c["q"].shape
    o, lse = np.zeros((t, h, d)), np.full((h, t), np.inf)
    bo, bl = np.zeros((t, h, d)), np.zeros((h, t))
    rows = np.zeros(t, bool)
    left, right = c["window"][0], 0 if c["causal"] else c["window"][1]
    g, sm = h // c["hk"], c["scale"]
    bias = 136 if dt == "bfloat16" else 72
    terms = 1 if dt == "bfloat16" else 2
    lib = rt.load_library()
    floats = lib.g950_paged_attention_int4_workspace(None, len(c["used"]), h, c["hk"], d, min(c["seqlen_q"], t), c["seqlen_k"]) // 4
    nrows = c["seqlen_q"] * g
    block = 16 if d == 256 or nrows <= 16 else 32
    parts = parts or max(1, floats // (len(c["used"]) * c["hk"] * -(-nrows // block) * block * (d + 2)))
    for b, used in enumerate(c["used"]):
        b0, b1 = int(c["cu"][b]), int(c["cu"][b + 1])
        n, keys = b1 - b0, min(int(used), c["table"].shape[1] * c["page"])
        j = np.arange(keys)
        at = c["table"][b, j // c["page"]]
        held = (at >= 0) & (at < c["pool"])
        if without is not None:
            held &= j // c["page"] != without
        at = np.where(held, at, 0)
        row = j % c["page"]
        part = min(keys, max(-(-(keys // 64 + 2) // parts), 4) * 64)
        m = 32 * -(-part // 128) + 32
        kc, vc = (ref.unpack(c[x][at, row]).astype(np.float64) - 8 for x in ("kc", "vc"))
        ks, vs = (c[x][at, row].astype(np.float64) for x in ("ks", "vs"))
        vc, vs = vc + codes, vs * np.array([scales, offsets])
        if zero:
            vc, vs = vc * 0, vs * 0
        for i in range(n):
            rows[b0 + i] = True
            p0 = i + int(used) - n
            vis = held.copy()
            if left >= 0:
                vis &= j >= p0 - left
            if right >= 0:
                vis &= j <= p0 + right + later
            if not vis.any():
                continue
            for kv in range(c["hk"]):
                hs = slice(kv * g, (kv + 1) * g)
                q = c["q"][b0 + i, hs].astype(np.float64)  # [g, d]
                s, off = ks[vis, kv, 0], ks[vis, kv, 1]
                x, qs = q @ kc[vis, kv].T, q.sum(-1, keepdims=True)
                z = (s * x + off * qs) * (sm * scale)
                top = z.max(-1, keepdims=True)
                e = np.exp(z - top)
                p = e / e.sum(-1, keepdims=True)
                v = vc[vis, kv] * vs[vis, kv, :1] + vs[vis, kv, 1:]
                if once:
                    ps = bf16_step(e * vs[vis, kv, 0])
                    o[b0 + i, hs] = (ps @ vc[vis, kv] + (e @ vs[vis, kv, 1])[:, None]) / e.sum(-1, keepdims=True)
                else:
                    o[b0 + i, hs] = p @ v
                lse[hs, b0 + i] = (top + np.log(e.sum(-1, keepdims=True)))[:, 0]
                if not bars:
                    continue
                q1 = np.abs(q).sum(-1, keepdims=True)
                qm = np.maximum(np.maximum(q, 0).sum(-1, keepdims=True), np.maximum(-q, 0).sum(-1, keepdims=True))
                eq = (d / 8 + 3) * U / 2 * q1
                ex = bias * (eq + U / 2 * np.abs(qs)) + U * d * (bias * qm + 8 * q1)
                er = sm * (s * ex + np.abs(off) * eq + 3 * U * (s * np.abs(x) + np.abs(off * qs))) + U * np.abs(z) + 2.0 ** -22
                er = np.abs(er)
                out = o[b0 + i, hs]
                spread = np.abs(v[None] - out[:, None])  # [g, keys, d]
                bo[b0 + i, hs] = (np.einsum("gk,gkd->gd", p * er, spread) * 1.05
                                  + 2.0 ** -(8 * terms) * (p * vs[vis, kv, 0]) @ np.abs(vc[vis, kv])
                                  + U * m * terms * 2 * 144 * (p @ vs[vis, kv, 0])[:, None]
                                  + U / 2 * (m + 64) * ((p @ np.abs(vs[vis, kv, 1]))[:, None] + np.abs(out))
                                  + HALF[dt] * np.abs(out) * 1.01 + TINY[dt])
                bl[hs, b0 + i] = er.max(-1) + 2.0 ** -20 * (1 + np.abs(lse[hs, b0 + i]) / 2)
    return (o, lse, rows, bo, bl) if bars else (o, lse, rows)


def check(want, o, lse, untouched=9.0):
    """o, lse (float64 arrays) of a call against ``attend``'s; rows that are not
    written hold ``untouched``."""
    wo, wl, rows, bo, bl = want
    bad = ~(np.abs(o - wo) <= bo)[rows]
    assert not bad.any(), ("o", int(bad.sum()), bad.size, float((np.abs(o - wo) / bo.clip(1e-300))[rows].max()))
    assert (o[~rows] == untouched).all() and (lse[:, ~rows] == untouched).all()
    gl, wl, bl = lse[:, rows], wl[:, rows], bl[:, rows]
    assert np.array_equal(gl == math.inf, wl == math.inf) and not np.isnan(gl).any()
    f = np.isfinite(wl)
    worst = np.abs(gl[f] - wl[f]) / bl[f]
    assert (worst <= 1).all(), ("lse", float(worst.max()))
