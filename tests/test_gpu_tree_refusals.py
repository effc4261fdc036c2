"""Trees whose drafts are refused in long runs, verified by several workgroups a sequence."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from compiler_amd import runtime as rt  # noqa: E402
from test_gpu_tree import VERIFY, verify_case, verify_check, verify_run  # noqa: E402

pytestmark = pytest.mark.gpu


def refused_case(ql, v, drafts, kinds, seed=0):
    """Trees nearly all of whose drafts are refused: numbers next to 1."""
    VERIFY["refusals"] = dict(ql=ql, v=v, kinds=kinds)
    c = verify_case("refusals", drafts, "float32", seed=seed)
    c["u"][:] = 1 - 2.0 ** -24
    return c


@pytest.mark.parametrize("drafts", ["drawn", "distinct"])
def test_more_refusals_than_32(drafts):
    """Roots with up to 299 children and trees behind them, several workgroups each."""
    for ql, v in (([61], 9001), ([300, 1, 0, 90], 4500), ([40, 129], 20011)):
        c = refused_case(ql, v, drafts, ["star", "tree"])
        got = verify_run(c, "float32")
        assert rt.module().last_kernel == "g950_verify_tree_f32_parts"
        verify_check(c, got)
        verify_check(c, verify_run(c, "float32", workspace=torch.empty(0, device="cuda")))


@pytest.mark.parametrize("drafts", ["drawn", "chosen"])
def test_the_largest_trees_keep_to_their_places(drafts):
    """1024 nodes, all children of the root: what lies behind the workspace stays as it is."""
    c = refused_case([1024, 7], 4100, drafts, ["star"])
    t, b = c["target"].shape[0], 2
    floats = rt.module().verify_tree_workspace(b, t, c["v"])
    room = torch.full((floats + 4096,), 7.0, device="cuda")
    verify_check(c, verify_run(c, "float32", workspace=room[:floats]))
    assert rt.module().last_kernel == "g950_verify_tree_f32_parts"
    assert (room[floats:] == 7.0).all()


def test_a_root_with_nothing_left():
    """Every draft refused and nothing left of p: one sum more than refusals."""
    c = refused_case([50], 8200, "drawn", ["star"])
    c["draft"][0] = np.maximum(c["target"][0] * 2, 2.0 ** -20)
    for ws in (None, torch.empty(0, device="cuda")):
        verify_check(c, verify_run(c, "float32", **({} if ws is None else {"workspace": ws})))
