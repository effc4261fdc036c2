"""What the paged conveniences do on the host before a call: no GPU, the module
and the launch stand in."""
import pytest

torch = pytest.importorskip("torch")

from compiler_amd import operators as ops  # noqa: E402
from compiler_amd import runtime as rt  # noqa: E402


class Module:
    device = 0

    @staticmethod
    def attention_int4_workspace(*sizes):
        return 96


@pytest.mark.parametrize("current,stream,floats", [(0, None, 96), (0x7F00, None, 96), (2, None, 0), (0, 2, 0), (0x7F00, 2, 0)])
def test_no_workspace_on_per_thread_streams(monkeypatch, current, stream, floats):
    """hipStreamPerThread (handle 2) names a stream of every thread, so memory that
    torch hands from one of its calls to the next may still be another
    thread's: also where it is torch's current stream."""
    got = []
    monkeypatch.setattr(rt, "module", Module)
    monkeypatch.setattr(rt, "_raw_stream", lambda device: current)
    monkeypatch.setattr(ops, "paged_attention_int4_kernel", lambda *a, **kw: got.append(a[10]))
    cache = torch.zeros((4, 16, 2, 32), dtype=torch.uint8)
    ops.paged_attention_int4(torch.zeros(3, 4, 64), cache, None, cache, None, None, torch.zeros(3), None, 1, 64,
                             **({} if stream is None else {"stream": stream}))
    assert got[0].shape == (floats,)
