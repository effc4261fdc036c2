"""That the bars of 4-bit paged attention tell right from wrong: results computed
wrongly on purpose (in float64, on the host), rounded as a kernel rounds them, are refused."""
import numpy as np
import pytest

pytest.importorskip("torch")

import paged_bars as bars  # noqa: E402
from oracle import paged as ref  # noqa: E402
from test_abi_paged import attend as host_attend  # noqa: E402
from test_gpu_paged_int4 import ATTEND  # noqa: E402

CASES = sorted(ATTEND) + sorted(bars.MORE)
WRONG = {
    "V is zero": dict(zero=True), "V's offsets ignored": dict(offsets=0.0), "V's codes one too high": dict(codes=1),
    "V's scales halved": dict(scales=0.5), "softmax scale 10% more": dict(scale=1.1), "softmax scale 10% less": dict(scale=0.9),
    "one key more": dict(later=1), "one key less": dict(later=-1), "a column of pages dropped": dict(without=1),
}
# what one key of thousands, or 64 of 16400, weighs less than the type's own roundings (where
# queries aim at such keys it is caught, below)
BELOW = {("ranges_d64", "one key more"), ("blocks_parts_d256", "one key more"), ("blocks_parts_d256", "one key less"), ("parts_window", "one key more"),
         ("parts_window_d256", "one key more"), ("parts_window_d256", "one key less"),
         ("short_beside_long", "one key more"), ("longest_parts", "one key less"),
         ("longest_parts", "a column of pages dropped")}
F16 = ["one_key", "tile_edges", "ranges_d64", "d256", "chunk_d64", "group3", "local_both", "fewer_keys_than_queries",
       "no_keys_no_queries", "page1", "wide_few_d64", "odd_d", "blocks_parts_window_d64", "parts_window"]
ONCE = ["one_key", "group3", "local_both", "fewer_keys_than_queries", "no_keys_no_queries", "page1", "wide_few_d64"]


def put(o, lse, rows, dt):
    """As a call leaves it: rounded, other rows untouched."""
    o, lse = ref.rounder(dt)(o).astype(np.float64), lse.astype(np.float32).astype(np.float64)
    o[~rows], lse[:, ~rows] = 9.0, 9.0
    return o, lse


def refuses(want, o, lse):
    try:
        bars.check(want, o, lse)
    except AssertionError:
        return True
    return False


def caught(c, dt, name, below=()):
    want = bars.attend(c, dt)
    o, lse = put(*want[:3], dt)
    bars.check(want, o, lse)
    for wrong, how in WRONG.items():
        got = bars.attend(c, dt, bars=False, **how)
        if np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]):
            continue  # (no such key, no such page)
        assert refuses(want, *put(*got, dt)) or (name, wrong) in below, wrong
    return want, o, lse


@pytest.mark.parametrize("name,dt", [(n, "bfloat16") for n in CASES] + [(n, "float16") for n in F16])
def test_wrong_results_are_refused(name, dt):
    c = bars.case(name, dt)
    want, o, lse = caught(c, dt, name, BELOW)
    assert refuses(want, o, np.where(want[2], lse + 0.05, lse))
    if name != "longest_parts":
        assert refuses(want, np.where(want[2][:, None, None], o * 1.1, o), lse)


@pytest.mark.parametrize("name", ["blocks_parts_d256", "parts_window", "parts_window_d256", "short_beside_long", "longest_parts",
                                  "ranges_d64", "blocks_parts_window_d64"])
def test_wrong_results_of_aimed_queries_are_refused(name):
    caught(bars.case(name, "bfloat16", aimed=True), "bfloat16", name)


@pytest.mark.parametrize("name", ONCE)
def test_float16_probabilities_in_one_term_are_refused(name):
    c = bars.case(name, "float16")
    want = bars.attend(c, "float16")
    assert refuses(want, *put(*bars.attend(c, "float16", bars=False, once=True), "float16"))


@pytest.mark.parametrize("dt", ["bfloat16", "float16"])
def test_every_kernel_has_a_case(dt):
    """The forms that the cases name are those that the launcher picks, and all it has."""
    import torch
    from compiler_amd import runtime as rt
    seen = set()
    for name in CASES:
        c = bars.case(name, dt)
        blocks = len(c["used"]) * c["hk"] * -(-c["seqlen_q"] * (c["h"] // c["hk"]) // 16)
        rc, kernel, err = host_attend(
            t=c["q"].shape[0], h=c["h"], hk=c["hk"], d=c["d"], pages=c["pool"], bs=c["page"], b=len(c["used"]),
            dt=rt.DT_BF16 if dt == "bfloat16" else rt.DT_F16, causal=c["causal"], scale=c["scale"], sk=c["seqlen_k"],
            sq=c["seqlen_q"], ws=blocks * 64 * 32 * (c["d"] + 2),
            page_table_ptr=dict(shape=list(c["table"].shape)))
        assert (rc, kernel) == (0, bars.kernel_of(name, c, dt)), (name, err)
        seen.add(kernel)
    t = "bf16" if dt == "bfloat16" else "f16"
    small = {f"g950_attn_int4_{t}_d{d}{f}" for d in (64, 128) for f in ("_r1", "_r2", "_r1w", "_r1_merge", "_r2_merge")}
    assert seen == small | {f"g950_attn_int4_{t}_d256{f}" for f in ("_r1", "_r1_merge")} | {"g950_attn_int4_general"}
