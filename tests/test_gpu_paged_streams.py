"""Streams that the paged conveniences are called on, and the memory they take there."""
import pytest

torch = pytest.importorskip("torch")

from compiler_amd import operators as ops  # noqa: E402
from compiler_amd import runtime as rt  # noqa: E402
from test_gpu_paged_int4 import attend_args, attend_case, check_attend  # noqa: E402

pytestmark = pytest.mark.gpu


def test_attend_on_the_per_thread_stream_as_current():
    """No workspace from the pool that all threads' per-thread streams share: one part."""
    c = attend_case("ranges", "bfloat16")
    args = attend_args(c, "bfloat16")
    o, lse = (torch.full(s, 9.0, device="cuda", dtype=dt) for s, dt in
              ((c["q"].shape, torch.bfloat16), ((c["h"], c["q"].shape[0]), torch.float32)))
    ops.paged_attention_int4(*args, scale=c["scale"], sync=True)
    assert rt.module().last_kernel.endswith("_merge")
    with torch.cuda.stream(torch.cuda.ExternalStream(2)):
        ops.paged_attention_int4(*args, scale=c["scale"], out=o, lse=lse, sync=True)
    assert rt.module().last_kernel.endswith("_r1")
    check_attend(c, "bfloat16", o, lse)
