"""Streams that the paged conveniences are called on, and the memory they take there."""
import pytest

torch = pytest.importorskip("torch")

from compiler_amd import operators as ops  # noqa: E402
from compiler_amd import runtime as rt  # noqa: E402
from own_streams import own_stream  # noqa: E402
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


def pool_of(t):
    """The stream whose pool a tensor's memory belongs to."""
    for seg in torch.cuda.memory_snapshot():
        if seg["address"] <= t.data_ptr() < seg["address"] + seg["total_size"]:
            return seg["stream"]
    raise AssertionError("no torch memory")


@pytest.mark.parametrize("as_handle", [False, True])
def test_outputs_come_from_the_calls_stream(as_handle):
    """Outputs of a call on another stream than torch's current one lie in that stream's
    pool: memory from the current one's could still be in use there.  Without a
    stream, in the current one's."""
    side = own_stream()
    bf = torch.bfloat16
    q, k = torch.randn(5, 4, 64, device="cuda").to(bf), torch.randn(5, 2, 64, device="cuda").to(bf)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    cos = torch.ones(8, 32, device="cuda")
    kc, ks = ops.int4_cache(2, 16, 2, 64, bf)
    vc, vs = ops.int4_cache(2, 16, 2, 64, bf)
    k16, v16 = (torch.zeros(2, 16, 2, 64, dtype=bf, device="cuda") for _ in range(2))
    lists = (torch.zeros(1, 1, dtype=torch.int32, device="cuda"), i32(0, 5), i32(5))
    x, w = torch.randn(7, 300, device="cuda"), torch.randn(300, device="cuda")
    torch.cuda.synchronize()
    for stream in (side.cuda_stream if as_handle else side, None):
        kw = dict(stream=stream, sync=True)
        q4, kv, vv = ops.paged_append_int4(q, k, k, cos, cos, kc, ks, vc, vs, *lists, values=True, **kw)
        outs = [q4, kv, vv, ops.paged_append(q, k, k, cos, cos, k16, v16, *lists, **kw),
                *ops.paged_attention_int4(q, kc, ks, vc, vs, *lists, 5, 5, **kw),
                *ops.block_norm(x, x, w, 1e-6, **kw)]
        torch.cuda.synchronize()
        want = torch.cuda.current_stream().cuda_stream if stream is None else side.cuda_stream
        assert [pool_of(t) for t in outs] == [want] * len(outs)
