"""Outputs that lie over inputs: what the paged operators and the norms around a
block take and refuse (g950_validate, no device).  Views are numpy views of host
buffers, which validation compares and never reads."""
import ctypes

import numpy as np
import pytest

from compiler_amd import runtime as rt

T, H, HK, D = 7, 8, 2, 64
OUTS = {"k_cache_ptr", "v_cache_ptr", "q_out_ptr", "k_out_ptr", "v_out_ptr", "k_scale_ptr", "v_scale_ptr", "Y", "N",
        "o_ptr", "softmax_lse_ptr", "workspace_ptr"}
CODES = {np.dtype(np.uint16): rt.DT_BF16, np.dtype(np.float32): rt.DT_F32, np.dtype(np.int32): rt.DT_INT32,
         np.dtype(np.uint8): rt.DT_UINT8}


def validate(op, views, scalars):
    names = sorted(views)
    arr, keep = (rt.View * len(names))(), []
    for i, n in enumerate(names):
        x = views[n]
        root = x
        while root.base is not None:
            root = root.base
        shape, strides = (ctypes.c_int64 * x.ndim)(*x.shape), (ctypes.c_int64 * x.ndim)(*x.strides)
        keep += [shape, strides]
        arr[i].data, arr[i].shape, arr[i].strides = x.ctypes.data, shape, strides
        arr[i].storage, arr[i].storage_size = root.ctypes.data, root.nbytes
        arr[i].dtype, arr[i].ndim, arr[i].flags = CODES[x.dtype], x.ndim, int(n in OUTS)
    sc = (rt.Scalar * len(scalars))(*[rt.scalar(s) for s in scalars])
    lib = rt.load_library()
    rc = lib.g950_validate(op, arr, len(names), sc, len(scalars))
    return rc, lib.g950_last_error().decode()


def half(*shape):
    return np.zeros(shape, np.uint16)


def append(four, **views):
    v = {"cos_ptr": np.zeros((50, D // 2), np.float32), "sin_ptr": np.zeros((50, D // 2), np.float32),
         "cu_seqlens_q_ptr": np.zeros(4, np.int32), "seqused_k_ptr": np.zeros(3, np.int32),
         "page_table_ptr": np.zeros((3, 4), np.int32), "q_ptr": half(T, H, D), "k_ptr": half(T, HK, D),
         "v_ptr": half(T, HK, D), "q_out_ptr": half(T, H, D)}
    for n in "kv":
        v[n + "_cache_ptr"] = np.zeros((9, 16, HK, D // 2), np.uint8) if four else half(9, 16, HK, D)
        if four:
            v[n + "_scale_ptr"], v[n + "_out_ptr"] = half(9, 16, HK, 2), half(T, HK, D)
    v.update(views)
    return validate(rt.OP_PAGED_APPEND_INT4 if four else rt.OP_PAGED_APPEND, v, [False])


def refused(got, *words):
    assert got[0] == rt.USAGE and all(w in got[1] for w in words), got


@pytest.mark.parametrize("four", [False, True])
def test_append_queries_over_inputs(four):
    qkv = half(T, H + 2 * HK, D)
    q, k, v = qkv[:, :H], qkv[:, H:H + HK], qkv[:, H + HK:]
    assert append(four, q_ptr=q, k_ptr=k, v_ptr=v)[0] == 0
    assert append(four, q_ptr=q, k_ptr=k, v_ptr=v, q_out_ptr=q)[0] == 0  # in place
    refused(append(four, q_ptr=q, k_ptr=k, v_ptr=v, q_out_ptr=qkv[:, 1:H + 1]), "q_out_ptr overlaps q_ptr")
    refused(append(four, q_ptr=qkv[:, 2 * HK:], k_ptr=k, v_ptr=v, q_out_ptr=qkv[:, 2 * HK:]), "q_out_ptr overlaps k_ptr")
    # the same start, other strides
    flat = half(2 * T * H * D)
    refused(append(four, q_ptr=flat[:T * H * D].reshape(T, H, D), q_out_ptr=flat.reshape(T, 2 * H, D)[:, ::2]),
            "q_out_ptr overlaps q_ptr")
    refused(append(four, q_ptr=flat[:T * H * D].reshape(T, H, D), q_out_ptr=flat[D:D + T * H * D].reshape(T, H, D)),
            "q_out_ptr overlaps q_ptr")
    # heads before tokens, backwards
    hm = half(H + 2 * HK, T, D).transpose(1, 0, 2)
    assert append(four, q_ptr=hm[:, :H], k_ptr=hm[:, H:H + HK], v_ptr=hm[:, H + HK:], q_out_ptr=hm[:, :H])[0] == 0
    refused(append(four, q_ptr=hm[:, :H], q_out_ptr=hm[::-1, :H]), "q_out_ptr overlaps q_ptr")
    # beside the inputs in one buffer: other heads of the rows, the other half of each head
    wide = half(T, 2 * H + 2 * HK, D)
    assert append(four, q_ptr=wide[:, :H], k_ptr=wide[:, H:H + HK], v_ptr=wide[:, -HK:], q_out_ptr=wide[:, H + HK:-HK])[0] == 0
    halves = half(T, H, 2 * D)
    assert append(four, q_ptr=halves[..., :D], q_out_ptr=halves[..., D:])[0] == 0
    rows = half(2 * T, H, D)
    assert append(four, q_ptr=rows[::2], q_out_ptr=rows[1::2])[0] == 0


def test_append_held_values_over_inputs():
    wide = half(T, H + 4 * HK, D)
    q, k, v, ko, vo = np.split(wide, [H, H + HK, H + 2 * HK, H + 3 * HK], 1)
    base = dict(q_ptr=q, k_ptr=k, v_ptr=v)
    assert append(True, **base, k_out_ptr=ko, v_out_ptr=vo)[0] == 0
    assert append(True, **base, k_out_ptr=half(0, 0, 0), v_out_ptr=half(0, 0, 0))[0] == 0
    refused(append(True, **base, k_out_ptr=k, v_out_ptr=vo), "k_out_ptr")
    refused(append(True, **base, k_out_ptr=v, v_out_ptr=vo), "k_out_ptr overlaps v_ptr")
    refused(append(True, **base, k_out_ptr=ko, v_out_ptr=k), "v_out_ptr overlaps k_ptr")
    refused(append(True, **base, k_out_ptr=ko, v_out_ptr=q[:, :HK]), "v_out_ptr overlaps q_ptr")
    refused(append(True, **base, k_out_ptr=wide[:, H + 1:H + 1 + HK], v_out_ptr=vo), "k_out_ptr overlaps k_ptr")
    refused(append(True, **base, k_out_ptr=ko, v_out_ptr=ko), "k_out_ptr overlaps v_out_ptr")
    out = half(T, H, D)
    refused(append(True, **base, q_out_ptr=out, k_out_ptr=out[:, :HK], v_out_ptr=vo), "k_out_ptr overlaps q_out_ptr")


def test_attend_over_queries():
    def attend(q, o):
        cache, pairs = np.zeros((9, 16, HK, D // 2), np.uint8), half(9, 16, HK, 2)
        v = {"cu_seqlens_q_ptr": np.zeros(4, np.int32), "seqused_k_ptr": np.zeros(3, np.int32),
             "page_table_ptr": np.zeros((3, 4), np.int32), "q_ptr": q, "o_ptr": o, "k_cache_ptr": cache,
             "v_cache_ptr": cache.copy(), "k_scale_ptr": pairs, "v_scale_ptr": pairs.copy(),
             "softmax_lse_ptr": np.zeros((H, T), np.float32), "workspace_ptr": np.zeros(0, np.float32)}
        return validate(rt.OP_PAGED_ATTENTION_INT4, v, [True, 0.1, 64, 3, -1, -1])
    qkv = half(T, 2 * H, D)
    assert attend(qkv[:, :H], half(T, H, D))[0] == attend(qkv[:, :H], qkv[:, :H])[0] == attend(qkv[:, :H], qkv[:, H:])[0] == 0
    refused(attend(qkv[:, :H], qkv[:, 1:H + 1]), "o_ptr overlaps q_ptr")
    rows = half(T + 1, H, D)
    refused(attend(rows[:T], rows[1:]), "o_ptr overlaps q_ptr")


def norm(**views):
    r, c = views["X"].shape
    v = {"G": half(0, 0), "W_post": half(c), "W_pre": half(c), "H": half(r, c), "Y": half(r, c), "N": half(r, c)}
    v.update(views)
    return validate(rt.OP_BLOCK_NORM, v, [1e-6, 0, 1.0])


@pytest.mark.parametrize("cols", [100, 40000])
def test_block_norm_over_inputs(cols):
    x, h, g = half(5, cols), half(5, cols), half(5, cols)
    for y in (x, h, g):
        for n in (x, h, g):
            if y is not n:
                assert norm(X=x, H=h, G=g, Y=y, N=n)[0] == 0
    refused(norm(X=x, H=h, Y=x, N=x), "N overlaps Y")
    wide = half(5, 2 * cols + 8)
    a, b = wide[:, :cols], wide[:, cols:2 * cols]
    assert norm(X=a, H=b)[0] == norm(X=a, H=h, Y=b)[0] == norm(X=a, H=b, Y=b, N=a)[0] == 0
    refused(norm(X=a, H=h, Y=wide[:, 1:cols + 1]), "Y overlaps X")
    refused(norm(X=a, H=b, N=wide[:, cols + 8:]), "N overlaps H")
    refused(norm(X=x, H=h, Y=wide[:, :cols], N=wide[:, 8:cols + 8]), "N overlaps Y")
    rows = half(6, cols)
    refused(norm(X=rows[:5], H=h, Y=rows[1:]), "Y overlaps X")
    refused(norm(X=x, H=h, Y=rows[:5], G=np.broadcast_to(rows[1], (5, cols))), "Y overlaps G")
    one = half(5, 1)
    assert norm(X=one, H=half(5, 1), Y=one)[0] == 0
