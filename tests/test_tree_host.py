"""What the conveniences of drafted trees do on the host before a call: no GPU, the module
and the launch stand in."""
import pytest

torch = pytest.importorskip("torch")

from compiler_amd import operators as ops  # noqa: E402
from compiler_amd import runtime as rt  # noqa: E402


class Module:
    device = 0
    asked = []

    @classmethod
    def attention_tree_workspace(cls, *sizes):
        cls.asked.append(sizes)
        return 96

    @classmethod
    def verify_tree_workspace(cls, *sizes):
        cls.asked.append(sizes)
        return 64


@pytest.fixture
def calls(monkeypatch):
    got = []
    monkeypatch.setattr(rt, "module", Module)
    monkeypatch.setattr(Module, "asked", [])
    monkeypatch.setattr(ops, "_new", lambda like, code, shape, stream: torch.empty(shape, dtype={
        0: like.dtype, rt.DT_F32: torch.float32, rt.DT_INT32: torch.int32}[code]))
    for name in ("paged_append_tree", "paged_attention_tree", "verify_tree", "paged_keep_path"):
        monkeypatch.setattr(ops, name + "_kernel", lambda *a, **kw: got.append(a))
    return got


CU = torch.zeros(3, dtype=torch.int32)


def attend(dtype=torch.bfloat16, **kw):
    cache = torch.zeros((4, 16, 2, 64), dtype=dtype)
    return ops.paged_attention_tree(torch.zeros((5, 4, 64), dtype=dtype), cache, cache, None, CU, None, None, 8, 100, **kw)


def verify(**kw):
    p = torch.zeros((5, 7))
    return ops.verify_tree(p, kw.pop("draft", p), torch.zeros(5, dtype=torch.int64), None, None, None, CU, 6, **kw)


@pytest.mark.parametrize("current,stream,given", [(0, None, True), (0x7F00, None, True), (2, None, False), (0, 2, False),
                                                  (0x7F00, 2, False)])
def test_no_workspace_on_per_thread_streams(monkeypatch, calls, current, stream, given):
    """hipStreamPerThread (handle 2) names a stream of every thread: no memory of torch's for it."""
    monkeypatch.setattr(rt, "_raw_stream", lambda device: current)
    kw = {} if stream is None else {"stream": stream}
    attend(**kw)
    verify(**kw)
    assert calls[0][9].shape == (96 if given else 0,) and calls[1][10].shape == (64 if given else 0,)


def test_sizes_asked_for(monkeypatch, calls):
    monkeypatch.setattr(rt, "_raw_stream", lambda device: 0)
    attend()
    verify()
    assert Module.asked == [(2, 4, 2, 64, 5, 100), (2, 5, 7)]  # (no more nodes than rows)
    attend(dtype=torch.float32)
    assert len(Module.asked) == 2 and calls[2][9].shape == (0,)
    ws = torch.zeros(7)
    attend(workspace=ws)
    verify(workspace=ws)
    assert len(Module.asked) == 2 and calls[3][9] is ws and calls[4][10] is ws


def test_outputs(monkeypatch, calls):
    monkeypatch.setattr(rt, "_raw_stream", lambda device: 0)
    o, lse = attend()
    assert o.shape == (5, 4, 64) and o.dtype == torch.bfloat16 and lse.shape == (4, 5) and lse.dtype == torch.float32
    assert calls[0][12] == 0.125 and calls[0][13] == -1
    path, count, token = verify(draft=None, distinct=True)
    assert path.shape == (2, 6) and path.dtype == count.dtype == torch.int32 and count.shape == token.shape == (2,)
    assert token.dtype == torch.int64 and calls[1][1].numel() == 0 and calls[1][11] is True
    k = torch.zeros((3, 2, 64))
    q = ops.paged_append_tree(None, k, k, None, None, None, None, None, CU, None, None)
    assert q.shape == (3, 0, 64)
    left = ops.paged_keep_path(None, None, None, CU, CU[:2], None, None)
    assert left.shape == (2,) and left.dtype == torch.int32
    kept = torch.zeros(2, dtype=torch.int32)
    assert ops.paged_keep_path(None, None, None, CU, CU[:2], None, None, out=kept) is kept
