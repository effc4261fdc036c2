"""Attention of drafted trees keeps to the workspace that it is given."""
import math

import pytest

torch = pytest.importorskip("torch")

from compiler_amd import runtime as rt  # noqa: E402
from test_gpu_tree import attend_case, attend_check, attend_run  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("share", [1, 2, 5])
@pytest.mark.parametrize("case", ["parts", "parts_d64", "parts_one", "parts_blocks", "longest_parts", "d256_parts",
                                  "part_edges", "many_parts", "wide_parts", "window_parts"])
def test_records_keep_to_their_places(case, share):
    """All of the workspace asked for, and parts of it: right, and what lies behind it stays."""
    c = attend_case(case, "bfloat16", seed=4)
    b, group = len(c["ql"]), c["h"] // c["hk"]
    floats = rt.module().attention_tree_workspace(b, c["h"], c["hk"], c["d"], min(c["seqlen_q"], c["q"].shape[0]),
                                                  c["seqlen_k"])
    assert floats % (min(c["seqlen_q"] * group, 128) * (c["d"] + 2)) == 0
    room = torch.full((floats + 65536,), math.nan, device="cuda")
    room[floats // share:] = 7.0
    attend_check(c, "bfloat16", *attend_run(c, "bfloat16", workspace=room[:floats // share]))
    assert ("merge" in rt.module().last_kernel) or share > 1
    assert (room[floats // share:] == 7.0).all()
