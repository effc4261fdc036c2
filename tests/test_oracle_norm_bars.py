"""That the bars of the norms around a block tell right from wrong: results computed
wrongly on purpose (in float64, on the host), rounded as a kernel rounds them, are refused."""
import numpy as np
import pytest

import norm_bars as bars
from oracle import paged as ref


def inputs(rows, cols, dt, gate, size=1.0, seed=0):
    rng = np.random.default_rng(seed)
    n = lambda *s: ref.rounder(dt)(rng.standard_normal(s).astype(np.float32) * size)  # noqa: E731
    return dict(x=n(rows, cols) * 2, h=n(rows, cols), w_pre=n(cols) / size, w_post=n(cols) / size,
                gate=n(rows, cols) / size if gate else None)


def put(x, dt):
    return ref.rounder(dt)(x.astype(np.float32)).astype(np.float64)


def refuses(want, y, n):
    try:
        bars.check(want, y, n)
    except AssertionError:
        return True
    return False


@pytest.mark.parametrize("dt", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("cols", [64, 1001, 4096, 40000])
def test_wrong_norms_are_refused(cols, dt):
    act, alpha = "tanh", 0.5
    i = inputs(4, cols, dt, True)
    want = bars.bounds(i, dt, act, alpha)
    y, n = put(want[0], dt), put(want[1], dt)
    bars.check(want, y, n)
    x, h, g = (i[k].astype(np.float64) for k in ("x", "h", "gate"))
    norm = lambda v, w, c=cols, e=1e-6: v / np.sqrt((v * v).sum(-1, keepdims=True) / c + e) * w  # noqa: E731
    step = {"float32": 1e-5, "bfloat16": 0.02, "float16": 0.003}[dt]  # a few of the type's steps, 84 in fp32
    wrong = {
        "one column more in the mean": norm(h, i["w_post"], cols + max(1, round(cols * step))),
        "no norm": h * i["w_post"],
        "no weight": norm(h, 1.0),
        "a column left out": norm(np.where(np.arange(cols) == cols - 1, 0, h), i["w_post"]),
    }
    for name, t in wrong.items():
        assert refuses(want, put(alpha * x + t * np.tanh(g), dt), n), name
    u = norm(h, i["w_post"])
    for name, v in {"sigmoid": alpha * x + u / (1 + np.exp(-g)), "no gate": alpha * x + u, "no scale": x + u * np.tanh(g),
                    "a gate off by some steps": alpha * x + u * np.tanh(g) * (1 + step)}.items():
        assert refuses(want, put(v, dt), n), name
    for name, v in {"of the block": norm(u, i["w_pre"]), "no weight": norm(want[0], 1.0),
                    "scale off": want[1] * (1 + step)}.items():
        assert refuses(want, y, put(v, dt)), name


@pytest.mark.parametrize("dt", ["bfloat16", "float16"])
def test_a_norm_of_the_rounded_y_is_refused(dt):
    i = inputs(40, 1000, dt, False)
    want = bars.bounds(i, dt)
    y, n = put(want[0], dt), put(want[1], dt)
    v = y / np.sqrt((y * y).mean(-1, keepdims=True) + 1e-6) * i["w_pre"]
    assert refuses(want, y, put(v, dt))


def test_another_epsilon_is_refused():
    """Rows whose squares are of epsilon's size."""
    for dt in ("float32", "bfloat16"):
        i = inputs(4, 1000, dt, False, size=2.0 ** -10)
        want = bars.bounds(i, dt)
        y, n = put(want[0], dt), put(want[1], dt)
        bars.check(want, y, n)
        for eps in (0.0, 2e-6):
            other = bars.bounds(i, dt, eps=eps)
            assert refuses(want, put(other[0], dt), n) and refuses(want, y, put(other[1], dt))
