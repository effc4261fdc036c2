"""Host-side contracts of the operators on drafted trees (g950_validate, no
device): what is taken, by which kernel, and what is refused."""
import pytest

from compiler_amd import runtime as rt
from test_abi_cpu import Args, validate

BF, F16, F32, I32, I64 = rt.DT_BF16, rt.DT_F16, rt.DT_F32, rt.DT_INT32, rt.DT_INT64


def call(op, views, scalars, change, outs):
    a = Args()
    for n in sorted(views):
        spec = dict(views[n], **change.get(n, {}))
        over = spec.pop("over", None)
        a.view(spec.pop("shape"), spec.pop("dtype"), output=spec.pop("output", n in outs), **spec)
        if over is not None:  # at the place of an earlier view
            shape, strides, dtype, output, _, _, size = a.specs[-1]
            data, storage = a.specs[sorted(views).index(over)][4:6]
            a.specs[-1] = (shape, strides, dtype, output, data, storage, size + (1 << 20))
    return validate(op, a, scalars)


def append(t=7, h=8, hk=2, d=128, r=None, pages=9, bs=16, b=3, dt=BF, **change):
    r = d if r is None else r
    v = {"cos_ptr": dict(shape=[50, r // 2], dtype=F32), "sin_ptr": dict(shape=[50, r // 2], dtype=F32),
         "cu_seqlens_q_ptr": dict(shape=[b + 1], dtype=I32), "seqused_k_ptr": dict(shape=[b], dtype=I32),
         "page_table_ptr": dict(shape=[b, 4], dtype=I32), "parent_ptr": dict(shape=[t], dtype=I32),
         "q_ptr": dict(shape=[t, h, d], dtype=dt), "q_out_ptr": dict(shape=[t, h, d], dtype=dt),
         "k_ptr": dict(shape=[t, hk, d], dtype=dt), "v_ptr": dict(shape=[t, hk, d], dtype=dt),
         "k_cache_ptr": dict(shape=[pages, bs, hk, d], dtype=dt), "v_cache_ptr": dict(shape=[pages, bs, hk, d], dtype=dt)}
    return call(rt.OP_PAGED_APPEND_TREE, v, [False], change, {"q_out_ptr", "k_cache_ptr", "v_cache_ptr"})


def attend(t=7, h=8, hk=2, d=128, pages=9, bs=16, b=3, dt=BF, scale=0.1, sk=64, sq=3, left=-1, ws=0, **change):
    v = {"cu_seqlens_q_ptr": dict(shape=[b + 1], dtype=I32), "seqused_k_ptr": dict(shape=[b], dtype=I32),
         "page_table_ptr": dict(shape=[b, 4], dtype=I32), "parent_ptr": dict(shape=[t], dtype=I32),
         "q_ptr": dict(shape=[t, h, d], dtype=dt), "o_ptr": dict(shape=[t, h, d], dtype=dt),
         "softmax_lse_ptr": dict(shape=[h, t], dtype=F32), "workspace_ptr": dict(shape=[ws], dtype=F32),
         "k_cache_ptr": dict(shape=[pages, bs, hk, d], dtype=dt), "v_cache_ptr": dict(shape=[pages, bs, hk, d], dtype=dt)}
    return call(rt.OP_PAGED_ATTENTION_TREE, v, [scale, sk, sq, left], change, {"o_ptr", "softmax_lse_ptr", "workspace_ptr"})


def verify(t=9, vocab=100, b=3, most=5, dt=F32, tk=I64, drawn=True, ws=0, **change):
    v = {"count_ptr": dict(shape=[b], dtype=I32), "cu_seqlens_q_ptr": dict(shape=[b + 1], dtype=I32),
         "draft_probs_ptr": dict(shape=[t, vocab] if drawn else [0, 0], dtype=dt), "next_ptr": dict(shape=[b], dtype=tk),
         "parent_ptr": dict(shape=[t], dtype=I32), "path_ptr": dict(shape=[b, most], dtype=I32),
         "target_probs_ptr": dict(shape=[t, vocab], dtype=dt), "tokens_ptr": dict(shape=[t], dtype=tk),
         "uniform_next_ptr": dict(shape=[b], dtype=F32), "uniform_ptr": dict(shape=[t], dtype=F32),
         "workspace_ptr": dict(shape=[ws], dtype=F32)}
    return call(rt.OP_VERIFY_TREE, v, [False], change, {"count_ptr", "next_ptr", "path_ptr", "workspace_ptr"})


def keep(b=3, pages=9, bs=16, hk=2, d=128, most=5, dt=BF, layers=None, **change):
    shape = [pages, bs, hk, d] if layers is None else [layers, pages, bs, hk, d]
    v = {"count_ptr": dict(shape=[b], dtype=I32), "cu_seqlens_q_ptr": dict(shape=[b + 1], dtype=I32),
         "k_cache_ptr": dict(shape=shape, dtype=dt), "page_table_ptr": dict(shape=[b, 4], dtype=I32),
         "path_ptr": dict(shape=[b, most], dtype=I32), "seqused_k_ptr": dict(shape=[b], dtype=I32),
         "seqused_out_ptr": dict(shape=[b], dtype=I32), "v_cache_ptr": dict(shape=shape, dtype=dt)}
    return call(rt.OP_PAGED_KEEP_PATH, v, [], change, {"k_cache_ptr", "v_cache_ptr", "seqused_out_ptr"})


def refused(got, code, what):
    rc, _, err = got
    assert rc == code and what in err, got


def test_append():
    for kw in (dict(), dict(h=0), dict(r=32), dict(r=0), dict(d=80, h=3, hk=3), dict(t=0), dict(dt=F16), dict(dt=F32),
               dict(pages=0), dict(bs=1), dict(d=300)):
        rc, name, err = append(**kw)
        assert rc == 0 and name.startswith("g950_kv_append_tree"), (kw, err)
    assert append()[1] == "g950_kv_append_tree_bf16_d128" and append(d=80)[1] == "g950_kv_append_tree_general"
    refused(append(parent_ptr=dict(shape=[6])), rt.USAGE, "int32 [tokens]")
    refused(append(parent_ptr=dict(dtype=I64)), rt.USAGE, "int32 [tokens]")
    refused(append(parent_ptr=dict(strides=[2])), rt.USAGE, "contiguous")
    refused(append(q_ptr=dict(shape=[6, 8, 128])), rt.USAGE, "disagree")
    refused(append(v_cache_ptr=dict(over="k_cache_ptr")), rt.USAGE, "overlaps")
    refused(append(q_out_ptr=dict(over="k_ptr")), rt.USAGE, "overlaps")
    assert append(q_ptr=dict(over="q_out_ptr"))[0] == 0
    refused(append(v_ptr=dict(over="k_cache_ptr")), rt.USAGE, "overlaps")


def test_attend():
    for kw in (dict(), dict(t=0), dict(d=64), dict(d=256), dict(d=80), dict(bs=10), dict(h=2), dict(h=64), dict(left=5),
               dict(sq=1024), dict(sq=0), dict(dt=F16), dict(dt=F32), dict(pages=0), dict(scale=0.0), dict(b=0, t=0)):
        rc, name, err = attend(**kw)
        assert rc == 0 and name.startswith("g950_attn_tree"), (kw, err)
    assert attend(o_ptr=dict(), q_ptr=dict(over="o_ptr"))[0] == 0
    refused(attend(o_ptr=dict(dtype=F16)), rt.USAGE, "share one dtype")
    refused(attend(dt=I32), rt.USAGE, "share one dtype")
    refused(attend(h=7), rt.USAGE, "query heads")
    refused(attend(d=257), rt.USAGE, "at most 256")
    refused(attend(sq=1025), rt.USAGE, "0 .. 1024")
    refused(attend(sq=-1), rt.USAGE, "0 .. 1024")
    refused(attend(sk=1 << 32), rt.USAGE, "out of range")
    refused(attend(scale=float("inf")), rt.USAGE, "finite")
    refused(attend(parent_ptr=dict(shape=[8])), rt.USAGE, "int32 [tokens]")
    refused(attend(softmax_lse_ptr=dict(shape=[7, 7])), rt.USAGE, "float32 [h, tokens]")
    refused(attend(k_cache_ptr=dict(dtype=F16)), rt.USAGE, "must be")
    refused(attend(v_cache_ptr=dict(shape=[9, 16, 2, 64])), rt.USAGE, "like the other caches")
    refused(attend(workspace_ptr=dict(dtype=BF)), rt.USAGE, "float32")
    refused(attend(q_ptr=dict(strides=[2048, 256, 2])), rt.USAGE, "contiguous")
    refused(attend(o_ptr=dict(strides=[0, 128, 1])), rt.USAGE, "repeats")
    refused(attend(o_ptr=dict(over="k_cache_ptr")), rt.USAGE, "overlaps")
    refused(attend(softmax_lse_ptr=dict(over="o_ptr")), rt.USAGE, "overlaps")
    refused(attend(ws=64, workspace_ptr=dict(over="q_ptr")), rt.USAGE, "overlaps")
    refused(attend(q_ptr=dict(over="o_ptr", strides=[2048, 128, 1])), rt.USAGE, "overlaps")


def test_verify():
    for kw in (dict(), dict(drawn=False), dict(dt=BF), dict(dt=F16), dict(tk=I32), dict(vocab=1), dict(most=1), dict(t=0),
               dict(b=0, t=0)):
        rc, name, err = verify(**kw)
        assert rc == 0 and name.startswith("g950_verify_tree"), (kw, err)
    refused(verify(dt=I32), rt.USAGE, "target_probs_ptr must be")
    refused(verify(draft_probs_ptr=dict(dtype=BF)), rt.USAGE, "draft_probs_ptr must be")
    refused(verify(draft_probs_ptr=dict(shape=[9, 99])), rt.USAGE, "draft_probs_ptr must be")
    refused(verify(vocab=0), rt.USAGE, "extent empty")
    refused(verify(most=0), rt.USAGE, "root")
    refused(verify(next_ptr=dict(dtype=I32)), rt.USAGE, "both be")
    refused(verify(tokens_ptr=dict(shape=[8])), rt.USAGE, "disagree")
    refused(verify(uniform_ptr=dict(dtype=BF)), rt.USAGE, "disagree")
    refused(verify(uniform_next_ptr=dict(shape=[4])), rt.USAGE, "disagree")
    refused(verify(path_ptr=dict(shape=[2, 5])), rt.USAGE, "disagree")
    refused(verify(cu_seqlens_q_ptr=dict(shape=[3])), rt.USAGE, "disagree")
    refused(verify(target_probs_ptr=dict(strides=[200, 2])), rt.USAGE, "contiguous")
    refused(verify(count_ptr=dict(strides=[0])), rt.USAGE, "repeats")
    refused(verify(path_ptr=dict(output=False)), rt.REJECTED, "output flag")
    refused(verify(path_ptr=dict(over="count_ptr")), rt.USAGE, "overlaps")
    refused(verify(parent_ptr=dict(over="next_ptr")), rt.USAGE, "overlaps")
    refused(verify(ws=64, workspace_ptr=dict(over="uniform_ptr")), rt.USAGE, "overlaps")
    refused(verify(workspace_ptr=dict(dtype=BF)), rt.USAGE, "float32")
    refused(verify(ws=64, workspace_ptr=dict(offset=1)), rt.USAGE, "16-byte")
    # as many workgroups as the workspace has places for
    assert verify(vocab=50000)[1] == "g950_verify_tree_f32"
    assert verify(vocab=50000, ws=9 * 4 + 3 * 64 * 2 - 1)[1] == "g950_verify_tree_f32"
    assert verify(vocab=50000, ws=9 * 4 + 3 * 64 * 2)[1] == "g950_verify_tree_f32_parts"
    assert verify(vocab=1000, ws=1 << 20)[1] == "g950_verify_tree_f32"


def test_keep():
    for kw, word in ((dict(), 16), (dict(dt=F32), 16), (dict(dt=F16, layers=3), 16), (dict(d=77), 2), (dict(d=78), 4),
                     (dict(dt=F32, d=77), 4), (dict(pages=0), 16), (dict(b=0), 16), (dict(most=0), 16), (dict(layers=0), 16)):
        rc, name, err = keep(**kw)
        assert rc == 0 and name == f"g950_kv_keep_w{word}", (kw, name, err)
    assert keep(k_cache_ptr=dict(strides=[4224, 264, 132, 1]))[1] == "g950_kv_keep_w4"
    assert keep(v_cache_ptr=dict(offset=1))[1] == "g950_kv_keep_w2"
    refused(keep(v_cache_ptr=dict(shape=[9, 16, 2, 64])), rt.USAGE, "differ in shape")
    refused(keep(v_cache_ptr=dict(dtype=F16)), rt.USAGE, "share one dtype")
    refused(keep(dt=I32), rt.USAGE, "share one dtype")
    refused(keep(v_cache_ptr=dict(shape=[1, 9, 16, 2, 128])), rt.USAGE, "must both be")
    refused(keep(k_cache_ptr=dict(shape=[16, 2, 128]), v_cache_ptr=dict(shape=[16, 2, 128])), rt.USAGE, "must both be")
    refused(keep(path_ptr=dict(shape=[2, 5])), rt.USAGE, "agree on b")
    refused(keep(count_ptr=dict(dtype=I64)), rt.USAGE, "int32")
    refused(keep(bs=0), rt.USAGE, "pages of no keys")
    refused(keep(hk=0), rt.USAGE, "extent empty")
    refused(keep(k_cache_ptr=dict(strides=[0, 256, 128, 1])), rt.USAGE, "repeats")
    refused(keep(k_cache_ptr=dict(strides=[8192, 512, 256, 2])), rt.USAGE, "contiguous")
    refused(keep(v_cache_ptr=dict(over="k_cache_ptr")), rt.USAGE, "overlaps")
    refused(keep(seqused_out_ptr=dict(over="seqused_k_ptr")), rt.USAGE, "overlaps")
    refused(keep(b=1 << 23, layers=40), rt.USAGE, "grid too large")


@pytest.mark.parametrize("op,nv,ns", [(rt.OP_PAGED_APPEND_TREE, 12, 1), (rt.OP_PAGED_ATTENTION_TREE, 10, 4),
                                      (rt.OP_VERIFY_TREE, 11, 1), (rt.OP_PAGED_KEEP_PATH, 8, 0)])
def test_arity(op, nv, ns):
    for v, s in ((nv - 1, ns), (nv, ns + 1)):
        a = Args()
        for _ in range(v):
            a.view([1], F32)
        refused(validate(op, a, [0] * s), rt.USAGE, "needs")
