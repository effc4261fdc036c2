"""Norms around a block with gate and residual on the GPU against the float64
oracle.  Both outputs round once (half a step of the type); the fp32 chain
before them is sums of c squares (relative c x 2^-24 at the worst, halved by the
root), and fewer than 16 roundings or ulps of exp and division: relative to the
largest term of y, not to y, where x and the block's output cancel."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from compiler_amd import operators as ops  # noqa: E402
from compiler_amd import runtime as rt  # noqa: E402
from oracle import paged as ref  # noqa: E402
from own_streams import own_stream  # noqa: E402

pytestmark = pytest.mark.gpu

T = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SHAPES = [(1, 1), (3, 7), (2, 64), (5, 256), (4, 1000), (3, 1001), (17, 3000), (2, 4096), (9, 4099), (600, 512), (2, 8192),
          (3, 16384), (2, 20001), (1, 40000), (0, 128)]


def dev(x, dt):
    return None if x is None else torch.from_numpy(np.ascontiguousarray(x)).to("cuda").to(T[dt])


def inputs(rows, cols, dt, gate=None, post=True, pre=True, seed=0):
    rng = np.random.default_rng(seed)
    rnd = ref.rounder(dt)
    n = lambda *s: rnd(rng.standard_normal(s).astype(np.float32))  # noqa: E731
    shape = {None: None, "scalar": (1, 1), "channel": (1, cols), "row": (rows, 1), "full": (rows, cols)}[gate]
    return dict(x=n(rows, cols) * 2, h=rnd(n(rows, cols) * 0.5 + 0.25), w_pre=n(cols) if pre else None,
                w_post=n(cols) if post else None, gate=n(*shape) if shape else None)


def check(i, dt, y, n, act="none", alpha=1.0, eps=1e-6):
    wy, wn = ref.block_norm(i["x"], i["h"], i["w_pre"], eps, i["w_post"], i["gate"], act, alpha)
    cols = i["x"].shape[1]
    size = np.abs(alpha * i["x"]) + np.abs(wy - alpha * i["x"])
    rel = (16 + cols / 2) * 2.0 ** -24
    half, tiny = torch.finfo(T[dt]).eps / 2, torch.finfo(T[dt]).smallest_normal * torch.finfo(T[dt]).eps
    gy = y.float().cpu().numpy()
    assert (np.abs(gy - wy) <= half * np.abs(wy) + rel * size + tiny).all(), np.abs(gy - wy).max()
    if wn is None:
        assert n is None
        return
    gn = n.float().cpu().numpy()
    r = np.abs(wn) / np.maximum(np.abs(wy), 1e-300)  # |w| / rms(y)
    assert (np.abs(gn - wn) <= half * np.abs(wn) + 2 * rel * (np.abs(wn) + r * size) + tiny).all(), np.abs(gn - wn).max()


def run(i, dt, **kw):
    y, n = ops.block_norm(dev(i["x"], dt), dev(i["h"], dt), dev(i["w_pre"], dt), 1e-6, w_post=dev(i["w_post"], dt),
                          gate=dev(i["gate"], dt), sync=True, **kw)
    return y, n


@pytest.mark.parametrize("dt", sorted(T))
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_block_norm(rows, cols, dt):
    i = inputs(rows, cols, dt)
    check(i, dt, *run(i, dt))


@pytest.mark.parametrize("dt", sorted(T))
@pytest.mark.parametrize("gate", ["scalar", "channel", "row", "full"])
@pytest.mark.parametrize("act", ["none", "sigmoid", "tanh"])
def test_block_norm_gates(gate, act, dt):
    for rows, cols in ((5, 3000), (3, 1001), (2, 20001)):
        i = inputs(rows, cols, dt, gate)
        if gate == "full":  # both ends of the activations
            i["gate"][0, :6] = [0.0, 60.0, -60.0, 0.17, -0.19, 1e-4]
            i["gate"] = ref.rounder(dt)(i["gate"])
        check(i, dt, *run(i, dt, gate_act=act, residual_scale=0.5), act=act, alpha=0.5)


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
@pytest.mark.parametrize("post,pre", [(False, True), (True, False), (False, False)])
def test_block_norm_parts_left_out(post, pre, dt):
    for rows, cols in ((5, 3000), (3, 1001), (2, 20001)):
        i = inputs(rows, cols, dt, "channel", post, pre)
        check(i, dt, *run(i, dt))


@pytest.mark.parametrize("cols", [256, 1001, 4096, 20001])
def test_block_norm_in_place_and_strided(cols):
    dt = "bfloat16"
    i = inputs(6, cols, dt)
    x, h = dev(i["x"], dt), dev(i["h"], dt)
    y, n = ops.block_norm(x, h, dev(i["w_pre"], dt), 1e-6, w_post=dev(i["w_post"], dt), out=x, norm_out=h, sync=True)
    assert y is x and n is h
    check(i, dt, y, n)
    wide = [torch.full((6, cols + 5), 7.0, device="cuda", dtype=T[dt]) for _ in range(4)]
    wide[0][:, 1:cols + 1], wide[1][:, 2:cols + 2] = dev(i["x"], dt), dev(i["h"], dt)
    y, n = wide[2][:, 3:cols + 3], wide[3][:, :cols]
    ops.block_norm(wide[0][:, 1:cols + 1], wide[1][:, 2:cols + 2], dev(i["w_pre"], dt), 1e-6, w_post=dev(i["w_post"], dt),
                   out=y, norm_out=n, sync=True)
    check(i, dt, y, n)
    assert (wide[2][:, :3] == 7).all() and (wide[2][:, cols + 3:] == 7).all() and (wide[3][:, cols:] == 7).all()


def test_block_norm_gate_of_other_strides():
    """A gate that is neither contiguous along the row nor one per row."""
    i = inputs(5, 3000, "bfloat16", "full")
    t = {k: dev(v, "bfloat16") for k, v in i.items()}
    y, n = ops.block_norm(t["x"], t["h"], t["w_pre"], 1e-6, w_post=t["w_post"], gate=t["gate"].t().contiguous().t(),
                          gate_act="tanh", sync=True)
    assert rt.module().last_kernel == "g950_block_norm_general"
    check(i, "bfloat16", y, n, act="tanh")


def test_block_norm_forms():
    for cols, form in ((100, "i1_b64"), (900, "i2_b64"), (2000, "i1_b256"), (4096, "i2_b256"), (8192, "i2_b512"),
                       (16000, "i2_b1024"), (30000, "i4_b1024")):
        i = inputs(2, cols, "float16", "full")
        check(i, "float16", *run(i, "float16", gate_act="sigmoid"), act="sigmoid")
        assert rt.module().last_kernel == f"g950_block_norm_f16_{form}_g1"


def test_block_norm_rows_keep_to_themselves():
    """A row of NaN, of infinities, of zeros: the others are as without it."""
    i = inputs(6, 3000, "bfloat16")
    want = [t.clone() for t in run(i, "bfloat16")]
    i["h"][1, 5], i["x"][2, 7], i["h"][3], i["x"][3] = np.nan, np.inf, 0.0, 0.0
    y, n = run(i, "bfloat16")
    for r in (0, 4, 5):
        assert torch.equal(y[r], want[0][r]) and torch.equal(n[r], want[1][r])
    assert torch.isnan(y[1]).all() and torch.isnan(n[1]).all()
    assert (y[3] == 0).all() and (n[3] == 0).all()
    assert torch.isinf(y[2, 7])


def test_block_norm_captured():
    i = inputs(33, 4096, "bfloat16", "full")
    t = {k: dev(v, "bfloat16") for k, v in i.items()}
    call = lambda: ops.block_norm(t["x"], t["h"], t["w_pre"], 1e-6, w_post=t["w_post"], gate=t["gate"],  # noqa: E731
                                  gate_act="sigmoid")
    want = [x.clone() for x in call()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=own_stream()):
        out = call()
    for _ in range(3):
        for x in out:
            x.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        assert all(torch.equal(a, b) for a, b in zip(call(), want))
    with rt.no_alloc():
        assert all(torch.equal(a, b) for a, b in zip(call(), want))


@pytest.mark.parametrize("cols", [1, 3])
def test_block_norm_rows_past_one_launch(cols):
    """2^26 - 1 workgroups of 64 threads fill a launch: the rows behind them."""
    rows = 2 ** 26 + 70
    x = torch.randn(rows, cols, device="cuda").bfloat16()
    h = torch.randn(rows, cols, device="cuda").bfloat16()
    gate = torch.randn(rows, 1, device="cuda").bfloat16()
    w = torch.randn(cols, device="cuda").bfloat16()
    y, n = ops.block_norm(x, h, w, 1e-6, w_post=w, gate=gate, sync=True)
    for s in (slice(0, 100), slice(2 ** 26 - 100, 2 ** 26 + 70)):
        some = [t[s].clone() for t in (x, h, gate)]
        sy, sn = ops.block_norm(some[0], some[1], w, 1e-6, w_post=w, gate=some[2], sync=True)
        assert torch.equal(y[s], sy) and torch.equal(n[s], sn)
