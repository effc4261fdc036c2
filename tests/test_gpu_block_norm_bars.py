"""Norms around a block on the GPU within the bars of norm_bars.py: every form, type,
gate and activation, also where epsilon counts."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import norm_bars as bars  # noqa: E402
from compiler_amd import operators as ops  # noqa: E402
from compiler_amd import runtime as rt  # noqa: E402
from oracle import paged as ref  # noqa: E402
from test_gpu_block_norm import SHAPES, dev, inputs, run  # noqa: E402

pytestmark = pytest.mark.gpu

TYPES = ["float32", "bfloat16", "float16"]


def check(i, dt, act=None, alpha=1.0):
    y, n = run(i, dt, gate_act=act, residual_scale=alpha)
    want = bars.bounds(i, dt, act or "none", alpha)
    bars.check(want, y.double().cpu().numpy(), None if n is None else n.double().cpu().numpy())
    again = run(i, dt, gate_act=act, residual_scale=alpha)
    assert torch.equal(y, again[0]) and (n is None or torch.equal(n, again[1]))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,cols", [s for s in SHAPES if s[0]])
def test_within_bars(rows, cols, dt):
    check(inputs(rows, cols, dt), dt)
    check(inputs(rows, cols, dt, "row", seed=1), dt, "sigmoid", 1.25)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("act", [None, "sigmoid", "tanh"])
@pytest.mark.parametrize("gate", ["scalar", "channel", "row", "full"])
def test_gates_within_bars(gate, act, dt):
    """Every way that gates are loaded, and values on either side of where tanh changes its form."""
    for rows, cols in ((5, 300), (5, 3000), (3, 1001), (2, 20001), (2, 40000)):
        i = inputs(rows, cols, dt, gate)
        if gate == "full":
            i["gate"][0] = ref.rounder(dt)(np.linspace(-0.3, 0.3, cols).astype(np.float32))
            i["gate"][1, :6] = ref.rounder(dt)(np.array([0.0, 60.0, -60.0, 0.18, -0.18, 1e-4], np.float32))
        check(i, dt, act, 0.5)


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
@pytest.mark.parametrize("cols", [100, 1000, 4096, 16000, 40000])
def test_small_rows_within_bars(cols, dt):
    """Squares of epsilon's size."""
    i = inputs(4, cols, dt, "full")
    for k in ("x", "h"):
        i[k] = i[k] * np.float32(2.0 ** -10)
    check(i, dt, "sigmoid")


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("post,pre", [(False, True), (True, False), (False, False)])
def test_parts_left_out_within_bars(post, pre, dt):
    for cols in (100, 3000, 40000):
        check(inputs(4, cols, dt, "channel", post, pre), dt, "tanh", 0.5)


@pytest.mark.parametrize("same", ["x", "h", "gate"])
@pytest.mark.parametrize("cols", [100, 4096, 20001, 40000])
def test_outputs_that_are_inputs(cols, same):
    """Y in the place of X, H or G, N in that of the next of them."""
    i = inputs(6, cols, "bfloat16", "full")
    t = {k: dev(v, "bfloat16") for k, v in i.items()}
    other = {"x": "h", "h": "gate", "gate": "x"}[same]
    y, n = ops.block_norm(t["x"], t["h"], t["w_pre"], 1e-6, w_post=t["w_post"], gate=t["gate"], gate_act="tanh",
                          out=t[same], norm_out=t[other], sync=True)
    assert y is t[same] and n is t[other] and (rt.module().last_kernel.endswith("general") == (cols == 40000))
    bars.check(bars.bounds(i, "bfloat16", "tanh"), y.double().cpu().numpy(), n.double().cpu().numpy())
