"""4-bit paged attention on the GPU within the bars of paged_bars.py, every
compiled form by name: blocks of query rows and parts of keys together, windows over parts,
queries that aim at single keys.  A call gives its bits again."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import paged_bars as bars  # noqa: E402
from compiler_amd import operators as ops  # noqa: E402
from compiler_amd import runtime as rt  # noqa: E402
from test_gpu_paged_int4 import ATTEND, attend_args, attend_run  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("aimed", [False, True])
@pytest.mark.parametrize("dt", ["bfloat16", "float16"])
@pytest.mark.parametrize("name", sorted(ATTEND) + sorted(bars.MORE))
def test_attend_within_bars(name, dt, aimed):
    c = bars.case(name, dt, aimed=aimed)
    args = attend_args(c, dt)
    o, lse = attend_run(c, dt, args)
    assert rt.module().last_kernel == bars.kernel_of(name, c, dt)
    bars.check(bars.attend(c, dt), o.double().cpu().numpy(), lse.double().cpu().numpy())
    for _ in range(2):
        again = attend_run(c, dt, args)
        assert torch.equal(again[0], o) and torch.equal(again[1], lse)


@pytest.mark.parametrize("name", ["blocks_parts", "chunk_d64", "parts_window", "wide_few", "rows33", "d256", "page10"])
def test_attend_in_the_place_of_its_queries(name):
    c = bars.case(name, "bfloat16")
    args = list(attend_args(c, "bfloat16"))
    args[0][c["cu"][-1]:] = 9.0
    lse = torch.full((c["h"], c["q"].shape[0]), 9.0, device="cuda")
    o, _ = ops.paged_attention_int4(*args, scale=c["scale"], causal=c["causal"], window=c["window"], out=args[0], lse=lse,
                                    sync=True)
    assert o is args[0]
    bars.check(bars.attend(c, "bfloat16"), o.double().cpu().numpy(), lse.double().cpu().numpy())


@pytest.mark.parametrize("dt", ["bfloat16", "float16"])
@pytest.mark.parametrize("name", ["blocks_parts", "blocks_parts_window_d64", "parts_window_d256", "wide_past_1024"])
def test_attend_in_one_part_within_bars(name, dt):
    """The same without a workspace: no parts, no second launch."""
    c = bars.case(name, dt)
    o, lse = attend_run(c, dt, workspace=torch.empty(0, device="cuda"))
    assert rt.module().last_kernel == bars.kernel_of(name, c, dt).replace("_merge", "")
    bars.check(bars.attend(c, dt, parts=1), o.double().cpu().numpy(), lse.double().cpu().numpy())


@pytest.mark.parametrize("name", ["blocks_parts", "blocks_parts_window_d64", "parts_window_d256"])
def test_attend_bad_pages_in_parts(name):
    """Pages outside the pool, at the edges of parts and across one."""
    c = bars.case(name, "bfloat16")
    c["table"][0, [0, 3, 4, 5, 11]] = [-1, c["pool"], -7, 1 << 30, -1]
    c["table"][1, :] = -1
    o, lse = attend_run(c, "bfloat16")
    assert rt.module().last_kernel == bars.kernel_of(name, c, "bfloat16")
    bars.check(bars.attend(c, "bfloat16"), o.double().cpu().numpy(), lse.double().cpu().numpy())
    b0, b1 = c["cu"][1:3]
    assert (o[b0:b1] == 0).all() and np.isposinf(lse[:, b0:b1].cpu().numpy()).all()
