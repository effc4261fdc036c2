"""Host-side contracts of the paged-cache operators and the norms around a
block (g950_validate, no device): what is taken, by which kernel, and what is
refused before anything is launched."""
import numpy as np
import pytest

from compiler_amd import runtime as rt
from oracle import paged as ref
from test_abi_cpu import Args, validate

BF, F16, F32, U8, I32 = rt.DT_BF16, rt.DT_F16, rt.DT_F32, rt.DT_UINT8, rt.DT_INT32

APPEND = ("cos_ptr", "cu_seqlens_q_ptr", "k_cache_ptr", "k_ptr", "page_table_ptr", "q_out_ptr", "q_ptr", "seqused_k_ptr",
          "sin_ptr", "v_cache_ptr", "v_ptr")
APPEND4 = tuple(sorted(APPEND + ("k_out_ptr", "v_out_ptr", "k_scale_ptr", "v_scale_ptr")))
ATTEND = ("cu_seqlens_q_ptr", "k_cache_ptr", "k_scale_ptr", "o_ptr", "page_table_ptr", "q_ptr", "seqused_k_ptr",
          "softmax_lse_ptr", "v_cache_ptr", "v_scale_ptr", "workspace_ptr")
OUT = {"k_cache_ptr", "v_cache_ptr", "q_out_ptr", "k_out_ptr", "v_out_ptr", "k_scale_ptr", "v_scale_ptr", "o_ptr",
       "softmax_lse_ptr", "workspace_ptr", "Y", "N"}


def args(names, views, change, attend=False):
    a = Args()
    for n in names:
        spec = dict(views[n])
        spec.update(change.get(n, {}))
        out = n in OUT and not (attend and n.startswith(("k_", "v_")))
        a.view(spec.pop("shape"), spec.pop("dtype"), output=spec.pop("output", out), **spec)
    return a


def append(four=False, t=7, h=8, hk=2, d=128, r=None, pages=9, bs=16, b=3, dt=BF, **change):
    r = d if r is None else r
    v = {"cos_ptr": dict(shape=[50, r // 2], dtype=F32), "sin_ptr": dict(shape=[50, r // 2], dtype=F32),
         "cu_seqlens_q_ptr": dict(shape=[b + 1], dtype=I32), "seqused_k_ptr": dict(shape=[b], dtype=I32),
         "page_table_ptr": dict(shape=[b, 4], dtype=I32), "q_ptr": dict(shape=[t, h, d], dtype=dt),
         "q_out_ptr": dict(shape=[t, h, d], dtype=dt), "k_ptr": dict(shape=[t, hk, d], dtype=dt),
         "v_ptr": dict(shape=[t, hk, d], dtype=dt), "k_out_ptr": dict(shape=[0, 0, 0], dtype=dt),
         "v_out_ptr": dict(shape=[0, 0, 0], dtype=dt)}
    for n in "kv":
        v[n + "_cache_ptr"] = dict(shape=[pages, bs, hk, d // 2 if four else d], dtype=U8 if four else dt)
        v[n + "_scale_ptr"] = dict(shape=[pages, bs, hk, 2], dtype=dt)
    return validate(rt.OP_PAGED_APPEND_INT4 if four else rt.OP_PAGED_APPEND, args(APPEND4 if four else APPEND, v, change),
                    [False])


def attend(t=7, h=8, hk=2, d=128, pages=9, bs=16, b=3, dt=BF, causal=True, scale=0.1, sk=64, sq=3, left=-1, right=-1,
           ws=0, **change):
    v = {"cu_seqlens_q_ptr": dict(shape=[b + 1], dtype=I32), "seqused_k_ptr": dict(shape=[b], dtype=I32),
         "page_table_ptr": dict(shape=[b, 4], dtype=I32), "q_ptr": dict(shape=[t, h, d], dtype=dt),
         "o_ptr": dict(shape=[t, h, d], dtype=dt), "softmax_lse_ptr": dict(shape=[h, t], dtype=F32),
         "workspace_ptr": dict(shape=[ws], dtype=F32)}
    for n in "kv":
        v[n + "_cache_ptr"] = dict(shape=[pages, bs, hk, d // 2], dtype=U8)
        v[n + "_scale_ptr"] = dict(shape=[pages, bs, hk, 2], dtype=dt)
    return validate(rt.OP_PAGED_ATTENTION_INT4, args(ATTEND, v, change, attend=True), [causal, scale, sk, sq, left, right])


def norm(rows=5, cols=256, dt=BF, act=0, **change):
    v = {"G": dict(shape=[0, 0], dtype=dt), "W_post": dict(shape=[cols], dtype=dt), "W_pre": dict(shape=[cols], dtype=dt)}
    for n in "HNXY":
        v[n] = dict(shape=[rows, cols], dtype=dt)
    return validate(rt.OP_BLOCK_NORM, args(sorted(v), v, change), [1e-6, act, 1.0])


def refused(got, code, what):
    rc, _, err = got
    assert rc == code and what in err, got


@pytest.mark.parametrize("four", [False, True])
def test_append_is_taken(four):
    for kw in (dict(), dict(h=0), dict(r=32), dict(r=0), dict(d=80, h=3, hk=3), dict(t=0), dict(dt=F16), dict(pages=0),
               dict(bs=1), dict(d=256)):
        rc, name, err = append(four, **kw)
        assert rc == 0 and name.startswith("g950_kv_append"), (kw, err)
    if not four:
        assert append(dt=F32)[0] == 0 and append(d=300)[0] == 0
    for r, general in ((128, False), (0, False), (16, False), (96, False), (32, False), (24, True), (2, True)):
        assert append(four, r=r)[1].endswith("_general") == general, r


@pytest.mark.parametrize("four", [False, True])
def test_append_refusals(four):
    op = lambda **kw: append(four, **kw)  # noqa: E731
    refused(op(k_ptr=dict(dtype=F16)), rt.USAGE, "share one dtype")
    refused(op(q_ptr=dict(shape=[6, 8, 128])), rt.USAGE, "disagree")
    refused(op(v_ptr=dict(shape=[7, 2, 64])), rt.USAGE, "disagree")
    refused(op(q_out_ptr=dict(shape=[7, 7, 128])), rt.USAGE, "q's shape")
    refused(op(q_ptr=dict(strides=[2048, 256, 2])), rt.USAGE, "contiguous")
    refused(op(sin_ptr=dict(shape=[49, 64])), rt.USAGE, "differ")
    refused(op(cos_ptr=dict(dtype=F16), sin_ptr=dict(dtype=F16)), rt.USAGE, "float32 or q's")
    refused(op(r=130), rt.USAGE, "turn")
    refused(op(cu_seqlens_q_ptr=dict(shape=[3])), rt.USAGE, "disagree on b")
    refused(op(page_table_ptr=dict(shape=[2, 4])), rt.USAGE, "disagree on b")
    refused(op(page_table_ptr=dict(dtype=rt.DT_INT64)), rt.USAGE, "int32")
    refused(op(v_cache_ptr=dict(shape=[8, 16, 2, 64 if four else 128])), rt.USAGE, "like the other caches")
    refused(op(k_cache_ptr=dict(shape=[9, 16, 3, 64 if four else 128])), rt.USAGE, "like the other caches")
    refused(op(k_cache_ptr=dict(dtype=F32)), rt.USAGE, "must be")
    refused(op(bs=0), rt.USAGE, "pages of no keys")
    refused(op(k_cache_ptr=dict(output=False)), rt.REJECTED, "output flag")
    refused(op(v_cache_ptr=dict(strides=[0, 128, 64, 1])), rt.USAGE, "repeats")
    refused(op(q_out_ptr=dict(strides=[0, 128, 1])), rt.USAGE, "repeats")
    refused(op(hk=0), rt.USAGE, "extent empty")
    if four:
        refused(op(dt=F32), rt.USAGE, "share one dtype")
        refused(op(d=258), rt.USAGE, "at most 256")
        refused(op(d=77), rt.USAGE, "even")
        refused(op(k_scale_ptr=dict(shape=[9, 16, 2, 1])), rt.USAGE, "like the other caches")
        refused(op(k_scale_ptr=dict(dtype=F32)), rt.USAGE, "must be")
        refused(op(k_out_ptr=dict(shape=[7, 2, 64])), rt.USAGE, "k's shape")
        refused(op(v_out_ptr=dict(shape=[7, 2, 128], dtype=F16)), rt.USAGE, "k's shape")


def test_attend_is_taken():
    for kw in (dict(), dict(t=0), dict(d=64), dict(d=256), dict(d=80), dict(bs=10), dict(bs=1), dict(h=2), dict(h=64),
               dict(left=5, right=9, causal=False), dict(sq=500), dict(sq=0), dict(dt=F16), dict(pages=0), dict(scale=0.0)):
        rc, name, err = attend(**kw)
        assert rc == 0 and name.startswith("g950_attn_int4"), (kw, err)


def test_attend_refusals():
    refused(attend(dt=F32), rt.USAGE, "share one dtype")
    refused(attend(o_ptr=dict(dtype=F16)), rt.USAGE, "share one dtype")
    refused(attend(h=7), rt.USAGE, "query heads")
    refused(attend(d=258), rt.USAGE, "at most 256")
    refused(attend(d=3), rt.USAGE, "even")
    refused(attend(sq=-1), rt.USAGE, "out of range")
    refused(attend(sk=1 << 32), rt.USAGE, "out of range")
    refused(attend(scale=float("nan")), rt.USAGE, "finite")
    refused(attend(scale=float("inf")), rt.USAGE, "finite")
    refused(attend(o_ptr=dict(shape=[7, 8, 64])), rt.USAGE, "q's shape")
    refused(attend(softmax_lse_ptr=dict(shape=[7, 8])), rt.USAGE, "float32 [h, tokens]")
    refused(attend(softmax_lse_ptr=dict(dtype=BF)), rt.USAGE, "float32 [h, tokens]")
    refused(attend(k_scale_ptr=dict(dtype=F16)), rt.USAGE, "must be")
    refused(attend(v_cache_ptr=dict(shape=[9, 8, 2, 64])), rt.USAGE, "like the other caches")
    refused(attend(seqused_k_ptr=dict(shape=[4])), rt.USAGE, "disagree on b")
    refused(attend(workspace_ptr=dict(dtype=BF)), rt.USAGE, "float32")
    refused(attend(workspace_ptr=dict(shape=[8], strides=[2])), rt.USAGE, "contiguous")
    refused(attend(o_ptr=dict(strides=[0, 128, 1])), rt.USAGE, "repeats")
    refused(attend(o_ptr=dict(output=False)), rt.REJECTED, "output flag")


def test_block_norm_is_taken_and_refused():
    for kw in (dict(), dict(cols=1), dict(cols=1001), dict(cols=100000), dict(rows=0), dict(dt=F32), dict(dt=F16),
               dict(W_post=dict(shape=[0])), dict(W_pre=dict(shape=[0]), N=dict(shape=[0, 0])),
               dict(G=dict(shape=[5, 256], strides=[0, 1]), act=1), dict(G=dict(shape=[5, 256], strides=[0, 0]), act=2)):
        rc, name, err = norm(**kw)
        assert rc == 0 and name.startswith("g950_block_norm"), (kw, err)
    refused(norm(cols=0), rt.USAGE, "empty row")
    refused(norm(act=3), rt.USAGE, "gate_act")
    refused(norm(act=1), rt.USAGE, "without G")
    refused(norm(G=dict(shape=[5, 255])), rt.USAGE, "X's shape")
    refused(norm(G=dict(shape=[5, 256], dtype=F32)), rt.USAGE, "X's shape")
    refused(norm(W_pre=dict(shape=[0])), rt.USAGE, "without W_pre")
    refused(norm(N=dict(shape=[0, 0])), rt.USAGE, "")
    refused(norm(W_post=dict(shape=[255])), rt.USAGE, "one entry per column")
    refused(norm(H=dict(dtype=F32)), rt.USAGE, "dtypes")
    refused(norm(H=dict(shape=[4, 256])), rt.USAGE, "shapes differ")
    refused(norm(Y=dict(strides=[0, 1])), rt.USAGE, "repeats")
    refused(norm(N=dict(strides=[0, 1])), rt.USAGE, "repeats")
    refused(norm(X=dict(strides=[512, 2])), rt.USAGE, "contiguous")


def test_block_norm_without_rows_takes_a_gate():
    for g in (dict(shape=[0, 256]), dict(shape=[0, 256], strides=[0, 1]), dict(shape=[0, 0])):
        assert norm(rows=0, act=1, G=g)[0] == 0


def test_attend_sizes_past_every_grid():
    big = dict(t=(1 << 27) - 1, h=16, hk=16, b=(1 << 27) - 2, sq=(1 << 27) - 1, sk=5000)
    refused(attend(**big), rt.USAGE, "grid too large")
    size = lambda *a: rt.load_library().g950_paged_attention_int4_workspace(None, *a)  # noqa: E731
    assert size(1 << 31, 65536, 65536, 128, 1 << 31, 1 << 31) == 0
    assert size(0, 8, 8, 128, 1, 5000) == size(1, 8, 3, 128, 1, 5000) == size(1, 8, 8, 80, 1, 5000) == 0
    assert size(1, 8, 8, 128, 1, 1000) == 0 < size(1, 8, 8, 128, 1, 5000)


def test_block_norm_longest_rows():
    """Positions of a row count on by 256 in 32 bits until they pass its end."""
    for dt in (BF, F32):
        long = dict(rows=1, dt=dt, W_post=dict(shape=[0]), W_pre=dict(shape=[0]), N=dict(shape=[0, 0]))
        assert norm(cols=2 ** 31 - 256, **long)[:2] == (0, "g950_block_norm_general")
        for cols in (2 ** 31 - 255, 2 ** 31 - 1, 2 ** 31):
            refused(norm(cols=cols, **long), rt.USAGE, "extent too large")


def test_grids_past_32_bits_of_work_items():
    """A launch counts its work-items (workgroups x threads) in 32 bits.  Norms take
    several launches then, appends the general kernel; attention is refused."""
    edge = 2 ** 26 - 1  # waves of one launch
    for rows in (edge, edge + 1, 2 ** 31 - 1):
        assert norm(rows=rows, cols=64)[:2] == (0, "g950_block_norm_bf16_i1_b64_g0")
        assert norm(rows=rows, cols=40000)[:2] == (0, "g950_block_norm_general")
    for four in (False, True):
        name = "g950_kv_append%s_bf16_d128" % ("_int4" if four else "")
        assert append(four, t=edge // 4 * 4, h=1, hk=1)[:2] == (0, name)
        assert append(four, t=edge // 4 * 4 + 1, h=1, hk=1)[:2] == (0, "g950_kv_append_general")
    assert attend(t=edge // 2, h=2, hk=2, d=80, sq=5)[:2] == (0, "g950_attn_int4_general")
    refused(attend(t=edge // 2 + 1, h=2, hk=2, d=80, sq=5), rt.USAGE, "grid too large")
    long = dict(t=2 ** 27 - 1, sq=2 ** 27 - 1, h=1, hk=1)
    assert attend(b=3, **long)[:2] == (0, "g950_attn_int4_bf16_d128_r2")
    refused(attend(b=4, **long), rt.USAGE, "grid too large")


# ------------------------------------------------------- the oracle's own pins
def test_oracle_quantize_bounds_and_special_rows():
    rng = np.random.default_rng(0)
    for dt, eps in (("bfloat16", 2.0 ** -8), ("float16", 2.0 ** -11)):
        x = rng.standard_normal((40, 64)).astype(np.float32) * 3 + 1
        c, s, o = ref.quantize(x, dt)
        v = ref.values(ref.pack(c), np.concatenate([s, o], -1))
        # half a step inside; at the ends as much more as 8 rounded scales and the offset move
        assert (np.abs(v - x) <= s * (0.5 + 8 * eps) + eps * np.abs(o) + 1e-6).all()
        x[0], x[1, 3], x[2, 5] = 2.5, np.inf, np.nan
        c, s, o = ref.quantize(x, dt)
        assert s[0] == 0 and o[0] == 2.5 and (c[0] == 8).all()
        assert np.isnan(s[1:3]).all() and np.isnan(o[1:3]).all() and np.isfinite(s[3:]).all()
    assert np.array_equal(ref.unpack(ref.pack(c)), c)


def test_oracle_rotation_is_a_rotation():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((5, 3, 16))
    a = rng.standard_normal((5, 8))
    for inter in (False, True):
        y = ref.rotate(x, np.cos(a), np.sin(a), inter)
        assert np.allclose((y ** 2).sum(-1), (x ** 2).sum(-1))
        assert np.allclose(ref.rotate(y, np.cos(a), -np.sin(a), inter), x)
    z = (x[..., 0::2] + 1j * x[..., 1::2]) * np.exp(1j * a)[:, None]
    y = ref.rotate(x, np.cos(a), np.sin(a), True)
    assert np.allclose(y[..., 0::2], z.real) and np.allclose(y[..., 1::2], z.imag)
    y = ref.rotate(x, np.cos(a[:, :2]), np.sin(a[:, :2]), False)  # the rest as it was
    assert np.array_equal(y[..., 4:], x[..., 4:]) and np.allclose(y[..., 0], x[..., 0] * np.cos(a[:, :1]) - x[..., 2] * np.sin(a[:, :1]))


def test_oracle_attention_of_equal_keys_is_the_mean_value():
    q, k = np.ones((3, 2, 4)), np.ones((6, 1, 4))
    v = np.arange(6.0)[:, None, None] * np.ones((6, 1, 4))
    o, lse, rows = ref.attention(q, [k], [v], [6], [0, 2], 0.5, -1, 0, 8)
    assert rows.tolist() == [True, True, False]
    assert np.allclose(o[0], np.arange(5).mean()) and np.allclose(o[1], 2.5) and np.allclose(lse[:, 1], 2 + np.log(6))
    o, lse, _ = ref.attention(q, [k], [v], [6], [0, 2], 0.5, 1, 0, 8)
    assert np.allclose(o[0], 3.5) and np.allclose(lse[:, 0], 2 + np.log(2))
    o, lse, _ = ref.attention(q, [k[:0]], [v[:0]], [0], [0, 2], 0.5, -1, 0, 8)
    assert (o == 0).all() and np.isinf(lse).all()


def test_oracle_block_norm():
    x = np.full((2, 8), 3.0)
    y, n = ref.block_norm(x, np.full((2, 8), -5.0), np.full(8, 2.0), 0.0, np.ones(8), np.full((2, 1), 2.0), "none", 0.5)
    assert np.allclose(y, 1.5 - 2.0) and np.allclose(n, -2.0)
    y, n = ref.block_norm(x, x, None, 0.0, None, np.zeros((1, 1)), "sigmoid")
    assert np.allclose(y, 4.5) and n is None
