"""Drafted trees beside the kernels of ordinary attention, on streams, in one captured step, and
verification where some workgroups' sums never come."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from compiler_amd import operators as ops  # noqa: E402
from compiler_amd import runtime as rt  # noqa: E402
from oracle import inputs, reference, tree as ref  # noqa: E402
from own_streams import own_stream  # noqa: E402
from test_gpu_paged_int4 import dev, host, rope  # noqa: E402
from test_gpu_paged_streams import pool_of  # noqa: E402
from test_gpu_tree import VERIFY, verify_case, verify_check, verify_run, tree_of  # noqa: E402
from test_gpu_varlen import BAR, run as varlen_run  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["bfloat16", "float16"])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("d", [64, 128])
def test_chains_are_the_varlen_kernels_causal_attention(d, page, dt):
    """Chains of up to 300 nodes over the varlen kernel's pages, lengths and queries: both kernels
    within that kernel's bar of its float64 oracle, so within two of each other, and rows without keys
    the same.  (The tree kernel's own bound is below the bar: roundings of the probabilities and of
    the output, 2^-8 sum p |V| each in bfloat16; |V| has a mean of 0.2 and is 1.2 at most, where one key has all of p
    and p = 1 is exact.)"""
    a, meta = inputs.varlen_case(batches=3, max_q=300, max_k=777, h=8, hk=2, d=d, paged=True, block_size=page, causal=True,
                                 window_right=0, seqused_trim=5)
    a = dict(a)
    a["seqused_k_ptr"] = a["seqused_k_ptr"].copy()
    a["seqused_k_ptr"][2] = 100  # fewer keys than rows: the first ones see none
    o, lse, eo, el = varlen_run(a, meta, dt)
    assert rt.module().last_kernel.startswith("g950_attn_fwd_") and "_varlen_p" in rt.module().last_kernel
    cu, used = a["cu_seqlens_q_ptr"], a["seqused_k_ptr"]
    shape = (-1, page, 2, d)
    parent = np.concatenate([np.arange(n) - 1 for n in np.diff(cu)]).astype(np.int32)
    mine, mine_lse = ops.paged_attention_tree(
        dev(a["q_ptr"].reshape(-1, 8, d), dt), dev(a["k_ptr"].reshape(shape), dt), dev(a["v_ptr"].reshape(shape), dt),
        dev(a["page_table_ptr"].reshape(3, -1)), dev(cu), dev(used), dev(parent), 300, 777, sync=True)
    assert rt.module().last_kernel.startswith("g950_attn_tree_" + ("bf16" if dt == "bfloat16" else "f16"))
    mine, mine_lse = host(mine).reshape(-1), mine_lse.cpu().numpy().reshape(-1)
    for got, want in ((mine, eo), (mine_lse, el)):
        ok, err = reference.isclose_verdict(got, want, BAR[dt], BAR[dt])
        assert ok, err
    assert np.array_equal(np.isinf(mine_lse), np.isinf(lse)) and np.isinf(lse).sum() == 8 * (int(cu[3] - cu[2]) - 100)
    assert (np.abs(mine - o) <= 2 * BAR[dt] * (1 + np.abs(eo))).all()


@pytest.mark.parametrize("as_handle", [False, True])
def test_outputs_come_from_the_calls_stream(as_handle):
    """Outputs of a call on another stream than torch's current one lie in that stream's pool, without
    a stream in the current one's; so do they where a stream is made the current one."""
    side = own_stream()
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    q, k = torch.randn(5, 4, 64, device="cuda").to(torch.bfloat16), torch.randn(5, 2, 64, device="cuda").to(torch.bfloat16)
    cos = torch.ones(40, 32, device="cuda")
    kc, vc = (torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    lists, parent = (ints(0, 1).view(1, 2), ints(0, 5), ints(20)), ints(-1, 0, 0, 1, 2)
    p = torch.softmax(torch.randn(5, 9000, device="cuda"), -1)
    tokens, u, last = torch.zeros(5, dtype=torch.int64, device="cuda"), torch.rand(5, device="cuda"), torch.rand(1, device="cuda")
    torch.cuda.synchronize()

    def outputs(**kw):
        path, count, token = ops.verify_tree(p, None, tokens, parent, u, last, lists[1], 5, **kw)
        return [path, count, token, ops.paged_append_tree(q, k, k, cos, cos, kc, vc, *lists, parent, **kw),
                *ops.paged_attention_tree(q, kc, vc, *lists, parent, 5, 20, **kw),
                ops.paged_keep_path(kc, vc, *lists, path, count, **kw)]
    here = torch.cuda.current_stream().cuda_stream
    for stream, want in ((side.cuda_stream if as_handle else side, side.cuda_stream), (None, here)):
        outs = outputs(stream=stream, sync=True)
        torch.cuda.synchronize()
        assert [pool_of(t) for t in outs] == [want] * len(outs)
    with torch.cuda.stream(side):
        outs = outputs()
    torch.cuda.synchronize()
    assert [pool_of(t) for t in outs] == [side.cuda_stream] * len(outs)


def test_outputs_on_another_stream_outlive_the_call():
    """What the current stream still reads is not handed on: outputs of calls on a stream, read by the
    current one while later calls on that stream take memory of the same sizes."""
    side = own_stream(1)
    c = [verify_case("large", "drawn", "float32", seed=s) for s in range(2)]
    give = [[dev(x[n]) for n in ("target", "draft", "tokens", "parent", "u", "last", "cu")] for x in c]
    want = [verify_run(x, "float32") for x in c]
    spin = torch.randn(4096, 4096, device="cuda")
    for i in range(12):
        out = ops.verify_tree(*give[i % 2], c[0]["most"], stream=side)
        torch.cuda.current_stream().wait_stream(side)
        for _ in range(4):
            torch.mm(spin, spin)       # the current stream is behind
        kept = [x.clone() for x in out]
        del out                        # their memory may go to the next call on the stream
        ops.verify_tree(*give[1 - i % 2], c[0]["most"], stream=side)
        torch.cuda.synchronize()
        for got, w in zip(kept, want[i % 2]):
            assert np.array_equal(got.cpu().numpy(), w)


def test_captured_step_of_all_four():
    """Append, attention, verification and the move of the path that it gives in one graph, two such
    graphs replayed in turn on new inputs with eager calls between them: the eager calls' bits, and the oracle's
    path and rows."""
    h, hk, d, vocab, page, b, n, dt = 8, 2, 128, 9000, 16, 3, 14, "bfloat16"
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    rng = np.random.default_rng(0)
    cos, sin = (dev(x) for x in rope(1200, d, rng))
    cu = ints([0, n, 2 * n, 3 * n])
    VERIFY["captured"] = dict(ql=[n] * b, v=vocab)

    def fresh(seed):
        rng, w = np.random.default_rng(seed), verify_case("captured", "drawn", "float32", seed=seed, sharp=4.0)
        t = b * n
        return dict(x=dev(rng.standard_normal((t, h + 2 * hk, d)).astype(np.float32), dt),
                    kc=dev(rng.standard_normal((b * 64, page, hk, d)).astype(np.float32), dt),
                    vc=dev(rng.standard_normal((b * 64, page, hk, d)).astype(np.float32), dt),
                    table=dev(rng.permutation(b * 64).reshape(b, 64).astype(np.int32)),
                    used=dev(rng.integers(n, 1000, b).astype(np.int32)),
                    parent=dev(np.concatenate([tree_of("tree", n, rng) for _ in range(b)]).astype(np.int32)),
                    target=dev(w["target"][:t]), draft=dev(w["draft"][:t]), tokens=dev(w["tokens"][:t]),
                    u=dev(w["u"][:t] * 0.5), last=dev(w["last"]))

    def step(s):
        q = ops.paged_append_tree(s["x"][:, :h], s["x"][:, h:h + hk], s["x"][:, h + hk:], cos, sin, s["kc"], s["vc"], s["table"],
                                  cu, s["used"], s["parent"])
        o, lse = ops.paged_attention_tree(q, s["kc"], s["vc"], s["table"], cu, s["used"], s["parent"], n, 1000)
        path, count, token = ops.verify_tree(s["target"], s["draft"], s["tokens"], s["parent"], s["u"], s["last"], cu, n)
        left = ops.paged_keep_path(s["kc"], s["vc"], s["table"], cu, s["used"], path, count)
        return q, o, lse, path, count, token, left
    slots, graphs = [fresh(1), fresh(2)], []
    step(fresh(3))
    torch.cuda.synchronize()
    for s in slots:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(s)
        graphs.append((g, out))
    accepted = 0
    for turn in range(4):
        given = [fresh(10 + 2 * turn + i) for i in range(2)]
        for s, new in zip(slots, given):
            for name, x in s.items():
                x.copy_(new[name])
        before = [[x["kc"].clone(), x["vc"].clone()] for x in given]
        for g, _ in graphs:
            g.replay()
        eager = [step(x) for x in given]
        torch.cuda.synchronize()
        for s, x, (_, out), want, old in zip(slots, given, graphs, eager, before):
            assert all(torch.equal(p, q) for p, q in zip(out, want))
            assert torch.equal(s["kc"], x["kc"]) and torch.equal(s["vc"], x["vc"])
            path, count, token = (y.cpu().numpy() for y in out[3:6])
            w = ref.verify(*(x[m].cpu().numpy() for m in ("target", "draft", "tokens", "parent", "u", "last")),
                           cu.cpu().numpy(), n, False)
            assert all(np.array_equal(p, q) for p, q in zip((path, count, token), w))
            used, table = x["used"].cpu().numpy(), x["table"].cpu().numpy()
            # the values, appended as they are, then moved
            v = host(old[1])
            for z in range(b):
                for i in range(n):
                    at = used[z] - n + i
                    v[table[z, at // page], at % page] = host(x["x"][z * n + i, h + hk:])
            v, left = ref.keep(v, cu.cpu().numpy(), used, table, path, count)
            assert np.array_equal(host(x["vc"]), v) and np.array_equal(out[6].cpu().numpy(), left)
            accepted += int(count.sum()) - b
    assert accepted > 0


# --------------------------------------------------- sums that never come
class VerifyArgs(ctypes.Structure):
    """The kernels' argument (g950_args.h)."""
    _fields_ = ([(n, ctypes.c_void_p) for n in ("target", "draft", "tokens", "parent", "u", "last", "cu", "path", "count", "next")]
                + [(n, ctypes.c_longlong) for n in ("t_row", "d_row", "path_z", "count_z", "next_z")]
                + [(n, ctypes.c_int) for n in ("T", "B", "V", "L", "token64", "distinct", "parts")]
                + [(n, ctypes.c_void_p) for n in ("px", "told")])


def launch(name, args, grid):
    """A kernel of the code object on torch's current stream."""
    hip = ctypes.CDLL(str(rt.LIB_PATH))  # (finds the HIP runtime that the library uses)
    torch.cuda.current_stream().synchronize()
    module, function = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipModuleLoad(ctypes.byref(module), str(rt.HSACO_PATH).encode()) == 0
    try:
        assert hip.hipModuleGetFunction(ctypes.byref(function), module, name.encode()) == 0
        params = (ctypes.c_void_p * 1)(ctypes.addressof(args))
        u = ctypes.c_uint
        assert hip.hipModuleLaunchKernel(function, u(grid), u(1), u(1), u(256), u(1), u(1), u(0),
                                         ctypes.c_void_p(torch.cuda.current_stream().cuda_stream), params, None) == 0
        torch.cuda.synchronize()
    finally:
        hip.hipModuleUnload(module)


@pytest.mark.parametrize("drafts", ["drawn", "distinct", "chosen"])
@pytest.mark.parametrize("run,told", [(1, ()), (1, (1, 2, 3, 4, 5, 6)), (1, (2, 5)), (1, (6,)), (2, (3, 4)), (4, ())])
def test_verification_without_some_workgroups(run, told, drafts):
    """Of a tree's seven workgroups the first `run` are launched; the sums of `told` are there, all others'
    never come.  Each wait ends by itself, what is missing is added up in place, and the path, its length, the
    token and the sums that are told are those of all seven."""
    parts = 7
    VERIFY["some"] = dict(ql=[40], v=20011)
    for seed in range(3):
        c = verify_case("some", drafts, "float32", seed=seed, sharp=3.0)
        c["u"][:] = np.maximum(c["u"], 0.7)
        c["last"][:] = 0.0  # the token: the first column with anything left, the first workgroup's
        t = c["target"].shape[0]
        ws = torch.zeros(4 * t + 2 * parts * max(t, 32), device="cuda")
        want = verify_run(c, "float32", workspace=ws)
        verify_check(c, want)
        assert rt.module().last_kernel == "g950_verify_tree_f32_parts"
        assert want[2][0] < 20011 // parts
        words = ws.view(torch.int64)
        sums = words[2 * t:2 * t + t * parts].view(t, parts)  # a row a round
        all_told = sums.clone()
        rounds = int((all_told[:40, 0] != -1).sum())
        assert rounds >= 1 and (all_told[:rounds] != -1).all() and (all_told[rounds:40] == -1).all()
        sums.fill_(-1)
        for p in told:
            sums[:, p] = all_told[:, p]
        give = {n: None if c[n] is None else dev(c[n]) for n in ("target", "draft", "tokens", "parent", "u", "last", "cu")}
        give["tokens"] = give["tokens"].to(torch.int64)
        out = dict(path=torch.full((1, c["most"]), 99, dtype=torch.int32, device="cuda"),
                   count=torch.full((1,), 99, dtype=torch.int32, device="cuda"), next=torch.full((1,), 99, device="cuda"))
        a = VerifyArgs(**{n: None if x is None else x.data_ptr() for n, x in {**give, **out}.items()}, t_row=c["v"],
                       d_row=c["v"], path_z=c["most"], count_z=1, next_z=1, T=t, B=1, V=c["v"], L=c["most"], token64=1,
                       distinct=int(drafts == "distinct"), parts=parts, px=words.data_ptr(), told=sums.data_ptr())
        launch("g950_verify_tree_f32_parts", a, run)
        for n, w in zip(("path", "count", "next"), want):
            assert np.array_equal(out[n].cpu().numpy(), w), n
        assert torch.equal(sums[:rounds, :run], all_told[:rounds, :run])
