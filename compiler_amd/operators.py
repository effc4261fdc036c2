"""The hot-path operators behind the reference kernels' own call signatures.

Each function takes the arguments of the reference Triton kernel it replaces
(same names, same meaning; pointer arguments are torch-ROCm device tensors,
runtime scalars are ints/floats) and launches the gfx950 kernel through the
C ABI.  Views and scalars are handed over in sorted argument-name order, the
layout the reference host packer produces (a100_support/native_io.py:74,81).

The triton launch grid and constexpr block sizes of the reference are not
arguments here: the launcher derives the grid from the view extents, and the
constexprs only shaped the reference's tiles.  The one constexpr with
semantics, attention's ``CAUSAL``, is a keyword argument.
"""
from __future__ import annotations

import functools
import math

import numpy as np

from . import runtime as rt


# sorted argument names of each call form: (op, views, scalars) names one form
_ORDER: dict = {}


def _launch(op, named_tensors: dict, outputs: set, named_scalars: dict, stream=None, sync=False,
            prepare=False):
    form = (op, len(named_tensors), len(named_scalars))
    order = _ORDER.get(form)
    if order is None:
        names = sorted(named_tensors)
        order = _ORDER[form] = (names, [n in outputs for n in names], sorted(named_scalars))
    names, outs, scalar_names = order
    tensors = [named_tensors[n] for n in names]
    scalars = [named_scalars[n] for n in scalar_names]
    if prepare:
        return rt.module().prepare(op, tensors, outs, scalars, stream=stream)
    return rt.module().launch(op, tensors, outs, scalars, stream=stream, sync=sync)


def _launch_sorted(op, tensors, outs, scalars, stream, sync, prepare):
    """The call with its tensors, output flags and scalars in sorted-name order
    (no dictionaries on the way); all tensors live on the current device."""
    mod = rt.module()
    here = mod.device
    for t in tensors:
        if t.get_device() != here:
            raise rt.G950Error(rt.USAGE, f"tensors on device {t.get_device()}, the current device is {here}")
    if prepare:
        return mod.prepare(op, tensors, outs, scalars, stream=stream)
    return mod.launch(op, tensors, outs, scalars, stream=stream, sync=sync)


def softmax_kernel(x_ptr, y_ptr, n_cols, *, stream=None, sync=False, prepare=False):
    """Row softmax (ops/suite/perf/softmax.py:21-32).  x/y: [rows, n_cols]."""
    return _launch(rt.OP_SOFTMAX, {"x_ptr": x_ptr, "y_ptr": y_ptr}, {"y_ptr"},
                   {"n_cols": n_cols}, stream, sync, prepare)


def softmax_kernel_inner(output_ptr, input_ptr, M, N, TILE_N=None, ONE_TILE_PER_CTA=None, *, stream=None,
                         sync=False, prepare=False):
    """Row softmax over flat buffers (ops/suite/dev/softmax_kernel_inner.py:12-72):
    row m is the N contiguous elements at input_ptr + m*N, written to
    output_ptr + m*N.  With both constexprs given they travel as scalars: the
    one-tile form (ONE_TILE_PER_CTA) with TILE_N < N normalises only the first
    TILE_N elements of each row and leaves the rest of the output untouched,
    as the reference's single masked tile does (:13-24)."""
    scalars = {"M": M, "N": N}
    if TILE_N is not None and ONE_TILE_PER_CTA is not None:
        scalars.update(ONE_TILE_PER_CTA=bool(ONE_TILE_PER_CTA), TILE_N=int(TILE_N))
    return _launch(rt.OP_SOFTMAX_INNER, {"input_ptr": input_ptr, "output_ptr": output_ptr}, {"output_ptr"},
                   scalars, stream, sync, prepare)


def layer_norm_forward_row(Y_ptr, Y_row_stride, X_ptr, X_row_stride, W_ptr, B_ptr, Mean_ptr, Mean_row_stride,
                           RSTD_ptr, RSTD_row_stride, n_rows, n_cols, eps, BLOCK_SIZE=None, *, stream=None,
                           sync=False, prepare=False):
    """Row LayerNorm forward (ops/suite/dev/layer_norm_forward_row.py:11-36):
    mean and rstd from sum(x) and sum(x^2) (E[x^2] - mean^2), x_hat rounded to
    X's dtype, Y = x_hat*W + B.  Buffers are flat, addressed by the row-stride
    scalars.  The reference loads BLOCK_SIZE columns unmasked, so BLOCK_SIZE
    must equal n_cols (a wider block would read the next row)."""
    if BLOCK_SIZE is not None and int(BLOCK_SIZE) != int(n_cols):
        raise rt.G950Error(rt.USAGE, "_layer_norm_forward_row: BLOCK_SIZE must equal n_cols (the reference "
                                     "loads BLOCK_SIZE columns without a mask)")
    return _launch(rt.OP_LAYERNORM_ROW, {"B_ptr": B_ptr, "Mean_ptr": Mean_ptr, "RSTD_ptr": RSTD_ptr, "W_ptr": W_ptr,
                                         "X_ptr": X_ptr, "Y_ptr": Y_ptr}, {"Y_ptr", "Mean_ptr", "RSTD_ptr"},
                   {"Mean_row_stride": Mean_row_stride, "RSTD_row_stride": RSTD_row_stride,
                    "X_row_stride": X_row_stride, "Y_row_stride": Y_row_stride,
                    "eps": np.float32(eps) if not isinstance(eps, np.generic) else eps,
                    "n_cols": n_cols, "n_rows": n_rows}, stream, sync, prepare)


# the reference's kernel name (a leading underscore in ops/suite/dev/layer_norm_forward_row.py:11)
_layer_norm_forward_row = layer_norm_forward_row


def gqa_kernel(Q, K, V, Out, stride_qh, stride_qm, stride_qk, stride_kh, stride_kn, stride_kk,
               stride_vh, stride_vk, stride_vn, stride_oh, stride_om, stride_on, H_Q, H_KV, N_CTX, scale,
               GROUP, HEAD_DIM=None, BLOCK_N=None, *, stream=None, sync=False, prepare=False):
    """Non-causal GQA attention forward (ops/suite/dev/gqa.py:20-59): Q/Out
    [Z, H_Q, N_CTX, HEAD_DIM], K/V [Z, H_KV, N_CTX, HEAD_DIM]; query head h
    reads KV head h // GROUP.  BLOCK_N only shaped the reference's tile."""
    head_dim = Q.shape[-1] if HEAD_DIM is None else HEAD_DIM
    return _launch(rt.OP_GQA, {"K": K, "Out": Out, "Q": Q, "V": V}, {"Out"},
                   {"GROUP": GROUP, "HEAD_DIM": head_dim, "H_KV": H_KV, "H_Q": H_Q, "N_CTX": N_CTX,
                    "scale": np.float32(scale) if not isinstance(scale, np.generic) else scale,
                    "stride_kh": stride_kh, "stride_kk": stride_kk, "stride_kn": stride_kn,
                    "stride_oh": stride_oh, "stride_om": stride_om, "stride_on": stride_on,
                    "stride_qh": stride_qh, "stride_qk": stride_qk, "stride_qm": stride_qm,
                    "stride_vh": stride_vh, "stride_vk": stride_vk, "stride_vn": stride_vn},
                   stream, sync, prepare)


def logsumexp_kernel(x_ptr, y_ptr, n_cols, *, stream=None, sync=False, prepare=False):
    """Row logsumexp (ops/suite/perf/logsumexp.py:16-38).  x: [rows, n_cols],
    y: [rows] (float32 in the reference): max over non-NaN entries plus
    log(sum(exp(x - max))); NaN for a row holding a NaN; an infinite max is
    returned as is."""
    return _launch(rt.OP_LOGSUMEXP, {"x_ptr": x_ptr, "y_ptr": y_ptr}, {"y_ptr"},
                   {"n_cols": n_cols}, stream, sync, prepare)


def dequantize_kernel(b_ptr, b_scale_ptr, fpb_ptr, K, N, stride_bk, stride_bn, stride_fpbk, stride_fpbn,
                      *, stream=None, sync=False, prepare=False):
    """int8 weight dequantisation fpb = b * b_scale[None, :]
    (ops/suite/perf/dequantize_matmul.py:28-43).  b: int8 [K, N]; b_scale [N]
    and fpb [K, N] share one float dtype; the stride scalars are element
    strides and must match the tensors'."""
    return _launch(rt.OP_DEQUANTIZE, {"b_ptr": b_ptr, "b_scale_ptr": b_scale_ptr, "fpb_ptr": fpb_ptr},
                   {"fpb_ptr"}, {"K": K, "N": N, "stride_bk": stride_bk, "stride_bn": stride_bn,
                                 "stride_fpbk": stride_fpbk, "stride_fpbn": stride_fpbn},
                   stream, sync, prepare)


_VARLEN_VIEWS = ("q_ptr", "k_ptr", "v_ptr", "o_ptr", "p_ptr", "softmax_lse_ptr", "cu_seqlens_q_ptr",
                 "cu_seqlens_k_ptr", "seqused_k_ptr", "philox_args", "alibi_slopes_ptr", "page_table_ptr")
_VARLEN_SCALARS = ("q_row_stride", "k_row_stride", "v_row_stride", "q_head_stride", "k_head_stride",
                   "v_head_stride", "o_row_stride", "o_head_stride", "q_batch_stride", "k_batch_stride",
                   "v_batch_stride", "o_batch_stride", "is_cu_seqlens_q", "is_cu_seqlens_k", "is_seqused_k",
                   "b", "bk", "h", "hk", "h_hk_ratio", "seqlen_q", "seqlen_k", "seqlen_q_rounded",
                   "seqlen_k_rounded", "d", "is_softcap", "softcap", "scale_softmax", "scale_softmax_log2",
                   "is_dropout", "p_dropout", "rp_dropout", "p_dropout_in_uint8_t", "return_softmax",
                   "is_causal", "is_local", "window_size_left", "window_size_right", "seqlenq_ngroups_swapped",
                   "is_paged", "is_alibi", "alibi_slopes_batch_stride", "total_q", "page_table_batch_stride",
                   "block_size", "k_page_stride")
# tile-shape constexprs of the reference kernel: accepted, no semantics here
_VARLEN_TILE = ("BLOCK_M", "BLOCK_N", "BLOCK_K", "KERNEL_NUM_WARPS", "PIPELINE_STAGES", "d_rounded")
_VARLEN_NAMES = frozenset(_VARLEN_VIEWS + _VARLEN_SCALARS + _VARLEN_TILE)


def flash_varlen_fwd_kernel(*, stream=None, sync=False, prepare=False, **args):
    """Variable-length attention forward (ops/suite/dev/flash_varlen_fwd_kernel.py:22-320),
    called with the reference kernel's argument names: cu_seqlens / fixed-length
    batches, seqused_k, GQA, causal and local windows, paged K/V.  Pointer
    arguments are device tensors (flattened to 1-D views); softcap, dropout,
    alibi, return_softmax and seqlenq_ngroups_swapped must be off."""
    unknown = args.keys() - _VARLEN_NAMES
    if unknown:
        raise TypeError(f"flash_varlen_fwd_kernel: unexpected arguments {sorted(unknown)}")
    missing = [n for n in _VARLEN_VIEWS + _VARLEN_SCALARS if n not in args]
    if missing:
        raise TypeError(f"flash_varlen_fwd_kernel: missing arguments {missing}")
    views = {n: args[n].reshape(-1) for n in _VARLEN_VIEWS}
    scalars = {n: args[n] for n in _VARLEN_SCALARS}
    return _launch(rt.OP_FLASH_VARLEN, views, {"o_ptr", "softmax_lse_ptr"}, scalars, stream, sync, prepare)


def dequant_matmul_kernel(a_ptr, b_ptr, b_scale_ptr, y_ptr, M, N, K, *, stream=None, sync=False, prepare=False):
    """dequantize_matmul fused into one GEMM: y = a . (b * b_scale[None, :])
    (ops/suite/perf/dequantize_matmul.py:28-43 then matmul.py:21-37).  a: [M, K]
    float, b: int8 logical [K, N] (pass ``bt.t()`` of a row-major [N, K] for the
    MFMA path), b_scale: [N] in a's dtype, y: [M, N]."""
    return _launch(rt.OP_DEQUANT_MATMUL, {"a_ptr": a_ptr, "b_ptr": b_ptr, "b_scale_ptr": b_scale_ptr,
                                          "y_ptr": y_ptr}, {"y_ptr"}, {"M": M, "N": N, "K": K},
                   stream, sync, prepare)


def rms_layernorm_forward_kernel(Y, Y_row_stride, X, X_row_stride, W, W_row_stride, r,
                                 r_row_stride, n_cols, eps, *, stream=None, sync=False, prepare=False):
    """RMSNorm forward (ops/suite/perf/fast_rms_layernorm.py:20-42)."""
    return _launch(rt.OP_RMS_LAYERNORM, {"Y": Y, "X": X, "W": W, "r": r}, {"Y", "r"},
                   {"Y_row_stride": Y_row_stride, "X_row_stride": X_row_stride,
                    "W_row_stride": W_row_stride, "r_row_stride": r_row_stride,
                    "n_cols": n_cols, "eps": np.float32(eps)}, stream, sync, prepare)


def layernorm_kernel(X, Y, W, B, Mean, Rstd, stride, N, eps, *, stream=None, sync=False, prepare=False):
    """LayerNorm forward with Mean/Rstd outputs
    (ops/suite/dev/fused_layernorm_triton.py:27-42)."""
    return _launch(rt.OP_LAYERNORM, {"X": X, "Y": Y, "W": W, "B": B, "Mean": Mean, "Rstd": Rstd},
                   {"Y", "Mean", "Rstd"}, {"stride": stride, "N": N, "eps": np.float32(eps)},
                   stream, sync, prepare)


def matmul_kernel(a_ptr, b_ptr, y_ptr, M, N, K, *, stream=None, sync=False, prepare=False):
    """Y = A.B with fp32 accumulation (ops/suite/perf/matmul.py:21-37).
    ``b_ptr`` is the logical [K, N] operand in either layout: column-major
    (K-contiguous, e.g. ``bt.t()`` of a row-major [N, K] tensor) or the
    reference's row-major [K, N], which the MFMA kernel reads as it lies
    (transposing LDS reads) from one 256 tile each way."""
    return _launch(rt.OP_MATMUL, {"a_ptr": a_ptr, "b_ptr": b_ptr, "y_ptr": y_ptr}, {"y_ptr"},
                   {"M": M, "N": N, "K": K}, stream, sync, prepare)


def matmul_i8_kernel(a_ptr, b_ptr, c_ptr, M, N, K, *, stream=None, sync=False, prepare=False):
    """8-bit integer dot -> int32, bit-exact modular accumulation, for the
    four signedness pairs of the i8 family (a100c/plan/tiles.py:118-131:
    int8/uint8 a_ptr and b_ptr in any combination)."""
    return _launch(rt.OP_MATMUL_I8, {"a_ptr": a_ptr, "b_ptr": b_ptr, "c_ptr": c_ptr}, {"c_ptr"},
                   {"M": M, "N": N, "K": K}, stream, sync, prepare)


def matmul_i8_dequant_kernel(a_ptr, b_ptr, sa_ptr, sb_ptr, y_ptr, M, N, K, *, stream=None,
                             sync=False, prepare=False):
    """int8 GEMM + dequant epilogue: y = bf16(acc * sa[m] * sb[n])
    (per-column rule of ops/suite/perf/dequantize_matmul.py:29-38)."""
    return _launch(rt.OP_MATMUL_I8_DEQUANT,
                   {"a_ptr": a_ptr, "b_ptr": b_ptr, "sa_ptr": sa_ptr, "sb_ptr": sb_ptr,
                    "y_ptr": y_ptr}, {"y_ptr"}, {"M": M, "N": N, "K": K}, stream, sync, prepare)


def attn_fwd_causal_kernel(q_ptr, k_ptr, v_ptr, out_ptr, Z, H, N_CTX, scale,
                           stride_qz, stride_qh, stride_qm, stride_qk,
                           stride_kz, stride_kh, stride_kn, stride_kk,
                           stride_vz, stride_vh, stride_vk, stride_vn,
                           stride_oz, stride_oh, stride_om, stride_on,
                           *, CAUSAL=True, lse_ptr=None, stream=None, sync=False,
                           prepare=False):
    """Attention forward (ops/suite/perf/attn_fwd_causal.py:20-55), with GQA
    when k/v carry fewer heads (ops/suite/dev/gqa.py:29) and the optional
    per-row logsumexp (ops/suite/dev/flash_varlen_fwd_kernel.py:309,318-320)."""
    tensors = {"q_ptr": q_ptr, "k_ptr": k_ptr, "v_ptr": v_ptr, "out_ptr": out_ptr}
    outputs = {"out_ptr"}
    op = rt.OP_ATTENTION
    if lse_ptr is not None:
        tensors["lse_ptr"] = lse_ptr
        outputs.add("lse_ptr")
        op = rt.OP_ATTENTION_LSE
    scalars = {"CAUSAL": bool(CAUSAL), "Z": Z, "H": H, "N_CTX": N_CTX,
               "scale": np.float32(scale) if not isinstance(scale, np.generic) else scale,
               "stride_qz": stride_qz, "stride_qh": stride_qh, "stride_qm": stride_qm,
               "stride_qk": stride_qk, "stride_kz": stride_kz, "stride_kh": stride_kh,
               "stride_kn": stride_kn, "stride_kk": stride_kk, "stride_vz": stride_vz,
               "stride_vh": stride_vh, "stride_vk": stride_vk, "stride_vn": stride_vn,
               "stride_oz": stride_oz, "stride_oh": stride_oh, "stride_om": stride_om,
               "stride_on": stride_on}
    return _launch(op, tensors, outputs, scalars, stream, sync, prepare)


def paged_append_kernel(q_ptr, k_ptr, v_ptr, cos_ptr, sin_ptr, q_out_ptr, k_cache_ptr, v_cache_ptr, page_table_ptr,
                        cu_seqlens_q_ptr, seqused_k_ptr, interleaved, *, stream=None, sync=False, prepare=False):
    """Position rotation of q and k, k and v appended to a paged cache
    (G950_OP_PAGED_APPEND; no reference counterpart).  q/q_out [tokens, h, d],
    k/v [tokens, hk, d], cos/sin [positions, r / 2] (the first r dims turn), caches
    [pages, block_size, hk, d], page_table [b, pages], cu_seqlens_q [b + 1],
    seqused_k [b] (keys of each sequence, the new ones among them)."""
    return _launch_sorted(rt.OP_PAGED_APPEND,
                          (cos_ptr, cu_seqlens_q_ptr, k_cache_ptr, k_ptr, page_table_ptr, q_out_ptr, q_ptr,
                           seqused_k_ptr, sin_ptr, v_cache_ptr, v_ptr),
                          (False, False, True, False, False, True, False, False, False, True, False), (interleaved,),
                          stream, sync, prepare)


def paged_append_int4_kernel(q_ptr, k_ptr, v_ptr, cos_ptr, sin_ptr, q_out_ptr, k_out_ptr, v_out_ptr, k_cache_ptr,
                             k_scale_ptr, v_cache_ptr, v_scale_ptr, page_table_ptr, cu_seqlens_q_ptr, seqused_k_ptr,
                             interleaved, *, stream=None, sync=False, prepare=False):
    """paged_append_kernel into a cache of 4 bits (G950_OP_PAGED_APPEND_INT4):
    codes uint8 [pages, block_size, hk, d / 2], scale and offset [pages,
    block_size, hk, 2] in the model's type.  k_out/v_out [tokens, hk, d]: the
    appended rows as the cache holds them (empty: not wanted)."""
    return _launch_sorted(rt.OP_PAGED_APPEND_INT4,
                          (cos_ptr, cu_seqlens_q_ptr, k_cache_ptr, k_out_ptr, k_ptr, k_scale_ptr, page_table_ptr,
                           q_out_ptr, q_ptr, seqused_k_ptr, sin_ptr, v_cache_ptr, v_out_ptr, v_ptr, v_scale_ptr),
                          (False, False, True, True, False, True, False, True, False, False, False, True, True, False,
                           True), (interleaved,), stream, sync, prepare)


def paged_attention_int4_kernel(q_ptr, k_cache_ptr, k_scale_ptr, v_cache_ptr, v_scale_ptr, page_table_ptr,
                                cu_seqlens_q_ptr, seqused_k_ptr, o_ptr, softmax_lse_ptr, workspace_ptr, seqlen_q, seqlen_k,
                                scale_softmax, is_causal, window_size_left, window_size_right, *, stream=None,
                                sync=False, prepare=False):
    """Attention over a paged cache of 4 bits (G950_OP_PAGED_ATTENTION_INT4; no
    reference counterpart): q/o [tokens, h, d], lse float32 [h, tokens], the
    cache and its lists as paged_append_int4_kernel fills them; windows as in
    flash_varlen_fwd_kernel, sizes below 0 without limit."""
    return _launch_sorted(rt.OP_PAGED_ATTENTION_INT4,
                          (cu_seqlens_q_ptr, k_cache_ptr, k_scale_ptr, o_ptr, page_table_ptr, q_ptr, seqused_k_ptr,
                           softmax_lse_ptr, v_cache_ptr, v_scale_ptr, workspace_ptr),
                          (False, False, False, True, False, False, False, True, False, False, True),
                          (is_causal, scale_softmax, seqlen_k, seqlen_q, window_size_left, window_size_right), stream,
                          sync, prepare)


def block_norm_kernel(X, H, W_post, G, W_pre, Y, N, eps, gate_act, residual_scale, *, stream=None, sync=False,
                      prepare=False):
    """The norms around a block with its gate and residual (G950_OP_BLOCK_NORM;
    no reference counterpart): u = H rsqrt(mean(H^2) + eps) W_post, Y =
    residual_scale X + act(G) u, N = Y rsqrt(mean(Y^2) + eps) W_pre, by rows.
    Empty W_post, G or W_pre (with N): that part is left out.  gate_act: 0
    none, 1 sigmoid, 2 tanh."""
    return _launch_sorted(rt.OP_BLOCK_NORM, (G, H, N, W_post, W_pre, X, Y),
                          (False, False, True, False, False, False, True), (eps, gate_act, residual_scale), stream, sync,
                          prepare)


def paged_append_tree_kernel(q_ptr, k_ptr, v_ptr, cos_ptr, sin_ptr, q_out_ptr, k_cache_ptr, v_cache_ptr, page_table_ptr,
                             cu_seqlens_q_ptr, seqused_k_ptr, parent_ptr, interleaved, *, stream=None, sync=False,
                             prepare=False):
    """paged_append_kernel for drafted trees (G950_OP_PAGED_APPEND_TREE; no
    reference counterpart): a sequence's tokens are the nodes of a tree, parent
    int32 [tokens] their parents within the sequence (below their own index; else
    none).  Node i goes to the cache row of position base + i and turns as position base + its
    depth, base = seqused_k - nodes."""
    return _launch_sorted(rt.OP_PAGED_APPEND_TREE,
                          (cos_ptr, cu_seqlens_q_ptr, k_cache_ptr, k_ptr, page_table_ptr, parent_ptr, q_out_ptr, q_ptr,
                           seqused_k_ptr, sin_ptr, v_cache_ptr, v_ptr),
                          (False, False, True, False, False, False, True, False, False, False, True, False),
                          (interleaved,), stream, sync, prepare)


def paged_attention_tree_kernel(q_ptr, k_cache_ptr, v_cache_ptr, page_table_ptr, cu_seqlens_q_ptr, seqused_k_ptr,
                                parent_ptr, o_ptr, softmax_lse_ptr, workspace_ptr, seqlen_q, seqlen_k, scale_softmax,
                                window_size_left, *, stream=None, sync=False, prepare=False):
    """Attention of drafted trees over a paged cache (G950_OP_PAGED_ATTENTION_TREE;
    no reference counterpart): q/o [tokens, h, d], lse float32 [h, tokens], the cache
    [pages, block_size, hk, d] and its lists as paged_append_tree_kernel fills them.
    A node sees the keys before the tree, its own and those above it."""
    return _launch_sorted(rt.OP_PAGED_ATTENTION_TREE,
                          (cu_seqlens_q_ptr, k_cache_ptr, o_ptr, page_table_ptr, parent_ptr, q_ptr, seqused_k_ptr,
                           softmax_lse_ptr, v_cache_ptr, workspace_ptr),
                          (False, False, True, False, False, False, False, True, False, True),
                          (scale_softmax, seqlen_k, seqlen_q, window_size_left), stream, sync, prepare)


def verify_tree_kernel(target_probs_ptr, draft_probs_ptr, tokens_ptr, parent_ptr, uniform_ptr, uniform_next_ptr,
                       cu_seqlens_q_ptr, path_ptr, count_ptr, next_ptr, workspace_ptr, distinct, *, stream=None,
                       sync=False, prepare=False):
    """Drafted trees verified against the target's probabilities
    (G950_OP_VERIFY_TREE; no reference counterpart): probabilities [tokens, v]
    after each node (draft: those that its children were drawn from, or empty), tokens and
    parent [tokens], uniform float32 [tokens] and [b]; path int32 [b, most], count int32
    [b] and the next token [b] come out."""
    return _launch_sorted(rt.OP_VERIFY_TREE,
                          (count_ptr, cu_seqlens_q_ptr, draft_probs_ptr, next_ptr, parent_ptr, path_ptr, target_probs_ptr,
                           tokens_ptr, uniform_next_ptr, uniform_ptr, workspace_ptr),
                          (True, False, False, True, False, True, False, False, False, False, True), (distinct,), stream,
                          sync, prepare)


def paged_keep_path_kernel(k_cache_ptr, v_cache_ptr, page_table_ptr, cu_seqlens_q_ptr, seqused_k_ptr, path_ptr, count_ptr,
                           seqused_out_ptr, *, stream=None, sync=False, prepare=False):
    """An accepted path's cache rows moved behind the keys before the tree
    (G950_OP_PAGED_KEEP_PATH; no reference counterpart): row base + i gets row base +
    path[b, i], i < count[b]; caches [pages, block_size, hk, d] or with the layers in
    front; seqused_out int32 [b] is base + count."""
    return _launch_sorted(rt.OP_PAGED_KEEP_PATH,
                          (count_ptr, cu_seqlens_q_ptr, k_cache_ptr, page_table_ptr, path_ptr, seqused_k_ptr,
                           seqused_out_ptr, v_cache_ptr), (False, False, True, False, False, False, True, True), (), stream,
                          sync, prepare)


def stream_copy(x, y, *, stream=None, sync=False, prepare=False):
    """y = x through the streaming-copy kernel (nontemporal 16-byte loads and
    stores, the row kernels' memory path); used to calibrate HBM counters."""
    return _launch(rt.OP_COPY, {"x": x, "y": y}, {"y"}, {}, stream, sync, prepare)


# ------------------------------------------------------ tensor conveniences
def softmax(x, out=None, **kw):
    import torch
    y = torch.empty_like(x) if out is None else out
    softmax_kernel(x, y, x.shape[-1], **kw)
    return y


def logsumexp(x, out=None, **kw):
    import torch
    y = torch.empty(x.shape[0], dtype=torch.float32, device=x.device) if out is None else out
    logsumexp_kernel(x, y, x.shape[-1], **kw)
    return y


def dequantize(b, scale, out=None, **kw):
    """b: int8 [K, N] tensor, scale: [N] float tensor -> b * scale in scale's dtype."""
    import torch
    y = torch.empty(b.shape, dtype=scale.dtype, device=b.device) if out is None else out
    dequantize_kernel(b, scale, y, b.shape[0], b.shape[1], b.stride(0), b.stride(1), y.stride(0),
                      y.stride(1), **kw)
    return y


def dequant_matmul(a, b, scale, out=None, **kw):
    """a [M,K] @ (b [K,N] int8 * scale[N]); pass ``bt.t()`` for a K-contiguous b."""
    import torch
    m, k = a.shape
    n = b.shape[1]
    y = torch.empty((m, n), dtype=a.dtype, device=a.device) if out is None else out
    dequant_matmul_kernel(a, b, scale, y, m, n, k, **kw)
    return y


def rmsnorm(x, w, eps, out=None, r=None, **kw):
    import torch
    y = torch.empty_like(x) if out is None else out
    r = torch.empty(x.shape[0], dtype=torch.float32, device=x.device) if r is None else r
    rms_layernorm_forward_kernel(y, y.stride(0), x, x.stride(0), w, 1, r, r.stride(0),
                                 x.shape[1], eps, **kw)
    return y, r


def layernorm(x, w, b, eps, out=None, mean=None, rstd=None, **kw):
    import torch
    y = torch.empty_like(x) if out is None else out
    mean = torch.empty(x.shape[0], dtype=torch.float32, device=x.device) if mean is None else mean
    rstd = torch.empty(x.shape[0], dtype=torch.float32, device=x.device) if rstd is None else rstd
    layernorm_kernel(x, y, w, b, mean, rstd, x.stride(0), x.shape[1], eps, **kw)
    return y, mean, rstd


def matmul(a, b, out=None, **kw):
    """a [M,K] @ b [K,N] (row-major b, or ``bt.t()`` for a K-contiguous one)."""
    import torch
    m, k = a.shape
    n = b.shape[1]
    y = torch.empty((m, n), dtype=a.dtype, device=a.device) if out is None else out
    matmul_kernel(a, b, y, m, n, k, **kw)
    return y


def attention(q, k, v, scale=None, causal=True, out=None, lse=None, **kw):
    import torch
    z, h, s, d = q.shape
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    o = torch.empty_like(q) if out is None else out
    if lse is None:
        lse = torch.empty((z, h, s), dtype=torch.float32, device=q.device)
    attn_fwd_causal_kernel(q, k, v, o, z, h, s, scale, *q.stride(), *k.stride(), *v.stride(),
                           *o.stride(), CAUSAL=causal, lse_ptr=lse, **kw)
    return o, lse


@functools.lru_cache(maxsize=None)
def _none(dtype, device, rank):
    """A view without elements: an argument left out."""
    import torch
    return torch.empty((0,) * rank, dtype=dtype, device=device)


def _torch_stream(stream):
    """torch's object for a call's ``stream`` (a Stream or a handle); None for
    hipStreamPerThread (handle 2), whose memory torch would hand on between threads."""
    import torch
    if hasattr(stream, "cuda_stream"):
        return None if stream.cuda_stream == 2 else stream
    if stream == 2:
        return None
    return torch.cuda.ExternalStream(stream) if stream not in (0, 1) else torch.cuda.default_stream()


def _on_stream(stream, make):
    """``make`` (torch.empty, torch.empty_like) for outputs of a call on ``stream``:
    memory that no other stream's pending work still uses, and that is not handed on
    before the current stream, where the caller may read it, is done with it."""
    import torch
    stream = _torch_stream(stream)
    if stream is None:
        return make
    here = torch.cuda.current_stream()

    def made(*args, **kw):
        with torch.cuda.stream(stream):
            t = make(*args, **kw)
        if stream.cuda_stream != here.cuda_stream and t.numel():
            t.record_stream(here)
        return t
    return made


def paged_append(q, k, v, cos, sin, k_cache, v_cache, page_table, cu_seqlens_q, seqused_k, interleaved=False,
                 out=None, **kw):
    """Appends k and v to the cache and returns the rotated q (``out=q``: in
    place; q may be None).  See paged_append_kernel."""
    import torch
    stream = kw.get("stream")
    empty_like = torch.empty_like if stream is None else _on_stream(stream, torch.empty_like)
    q = k.new_empty((k.shape[0], 0, k.shape[2])) if q is None else q
    out = empty_like(q, memory_format=torch.contiguous_format) if out is None else out
    paged_append_kernel(q, k, v, cos, sin, out, k_cache, v_cache, page_table, cu_seqlens_q, seqused_k,
                        bool(interleaved), **kw)
    return out


def int4_cache(pages, block_size, heads, dim, dtype, device="cuda"):
    """An empty 4-bit K or V cache: codes uint8 [pages, block_size, heads, dim / 2]
    and scales dtype [pages, block_size, heads, 2], a page holding each head's
    rows together (the layout the attention kernels stream best)."""
    import torch
    codes = torch.zeros((pages, heads, block_size, dim // 2), dtype=torch.uint8, device=device)
    scale = torch.zeros((pages, heads, block_size, 2), dtype=dtype, device=device)
    return codes.transpose(1, 2), scale.transpose(1, 2)


def paged_append_int4(q, k, v, cos, sin, k_cache, k_scale, v_cache, v_scale, page_table, cu_seqlens_q, seqused_k,
                      interleaved=False, out=None, values=False, k_out=None, v_out=None, **kw):
    """paged_append into a cache of 4 bits (int4_cache).  Returns the rotated q
    and, with ``values`` (or k_out / v_out given), the appended keys and values
    as the cache holds them; else None for both."""
    import torch
    stream = kw.get("stream")
    empty_like = torch.empty_like if stream is None else _on_stream(stream, torch.empty_like)
    q = k.new_empty((k.shape[0], 0, k.shape[2])) if q is None else q
    out = empty_like(q, memory_format=torch.contiguous_format) if out is None else out
    if values:
        k_out = empty_like(k, memory_format=torch.contiguous_format) if k_out is None else k_out
        v_out = empty_like(v, memory_format=torch.contiguous_format) if v_out is None else v_out
    none = _none(k.dtype, k.device, 3)
    paged_append_int4_kernel(q, k, v, cos, sin, out, none if k_out is None else k_out, none if v_out is None else v_out,
                             k_cache, k_scale, v_cache, v_scale, page_table, cu_seqlens_q, seqused_k, bool(interleaved),
                             **kw)
    return out, k_out, v_out


def _workspace(floats, like, stream):
    """Memory for one call on ``stream`` (None: the current one), which torch
    may hand on when the call returns: to later work of that stream.  None for
    hipStreamPerThread (handle 2, also as torch's current stream), which names a
    stream of every thread."""
    import torch
    if stream is None:
        per_thread = rt._raw_stream(rt.module().device) == 2
    else:
        stream = _torch_stream(stream)
        per_thread = stream is None
    if stream is None or not floats:
        return torch.empty(0 if per_thread else floats, dtype=torch.float32, device=like.device)
    with torch.cuda.stream(stream):
        return torch.empty(floats, dtype=torch.float32, device=like.device)


def paged_attention_int4(q, k_cache, k_scale, v_cache, v_scale, page_table, cu_seqlens_q, seqused_k, seqlen_q, seqlen_k,
                         scale=None, causal=True, window=(-1, -1), out=None, lse=None, workspace=None, **kw):
    """Attention of q over a paged cache of 4 bits; seqlen_q is the most
    queries, seqlen_k the most keys of a sequence.  Returns o and lse [h, tokens].
    The workspace (float32) comes from torch's allocator, on the call's stream,
    unless given."""
    import torch
    t, h, d = q.shape
    seqlen_q, seqlen_k = int(seqlen_q), int(seqlen_k)
    stream = kw.get("stream")
    if out is None:
        o = (torch.empty_like if stream is None else _on_stream(stream, torch.empty_like))(
            q, memory_format=torch.contiguous_format)
    else:
        o = out
    if lse is None:
        lse = (torch.empty if stream is None else _on_stream(stream, torch.empty))(
            (h, t), dtype=torch.float32, device=q.device)
    if workspace is None:
        workspace = _workspace(rt.module().attention_int4_workspace(
            cu_seqlens_q.shape[0] - 1, h, k_cache.shape[2], d, min(seqlen_q, t), seqlen_k), q, stream)
    paged_attention_int4_kernel(q, k_cache, k_scale, v_cache, v_scale, page_table, cu_seqlens_q, seqused_k, o, lse,
                                workspace, seqlen_q, seqlen_k, 1.0 / math.sqrt(d) if scale is None else float(scale),
                                bool(causal), int(window[0]), int(window[1]), **kw)
    return o, lse


def _new(like, code, shape, stream):
    """torch.empty of ``shape`` on like's device, its dtype by code (0: like's), for an output
    of a call on ``stream``."""
    if stream is None:
        t = (rt._packer or rt._load_packer()).empty(like, code, *shape)
        if t is not None:
            return t
    import torch
    dtype = {0: like.dtype, rt.DT_F32: torch.float32, rt.DT_INT32: torch.int32}[code]
    return (torch.empty if stream is None else _on_stream(stream, torch.empty))(shape, dtype=dtype, device=like.device)


def _room(floats, like, stream):
    """_workspace, from native code on the current stream."""
    if stream is None and rt._raw_stream(rt.module().device) != 2:
        return _new(like, rt.DT_F32, (floats,), None)
    return _workspace(floats, like, stream)


def paged_append_tree(q, k, v, cos, sin, k_cache, v_cache, page_table, cu_seqlens_q, seqused_k, parent,
                      interleaved=False, out=None, **kw):
    """paged_append for drafted trees: ``parent`` holds each token's parent within its
    sequence.  See paged_append_tree_kernel."""
    q = k.new_empty((k.shape[0], 0, k.shape[2])) if q is None else q
    out = _new(q, 0, q.shape, kw.get("stream")) if out is None else out
    paged_append_tree_kernel(q, k, v, cos, sin, out, k_cache, v_cache, page_table, cu_seqlens_q, seqused_k, parent,
                             bool(interleaved), **kw)
    return out


def paged_attention_tree(q, k_cache, v_cache, page_table, cu_seqlens_q, seqused_k, parent, seqlen_q, seqlen_k, scale=None,
                         window_left=-1, out=None, lse=None, workspace=None, **kw):
    """Attention of drafted trees over a paged cache; seqlen_q is the most nodes (up
    to 1024), seqlen_k the most keys of a sequence.  Returns o and lse [h,
    tokens].  The workspace (float32) comes from torch's allocator, on the
    call's stream, unless given."""
    t, h, d = q.shape
    seqlen_q, seqlen_k = int(seqlen_q), int(seqlen_k)
    stream = kw.get("stream")
    o = _new(q, 0, (t, h, d), stream) if out is None else out
    lse = _new(q, rt.DT_F32, (h, t), stream) if lse is None else lse
    if workspace is None:
        floats = 0
        if q.element_size() == 2:
            floats = rt.module().attention_tree_workspace(cu_seqlens_q.shape[0] - 1, h, k_cache.shape[2], d,
                                                          min(seqlen_q, t), seqlen_k)
        workspace = _room(floats, q, stream)
    paged_attention_tree_kernel(q, k_cache, v_cache, page_table, cu_seqlens_q, seqused_k, parent, o, lse, workspace,
                                seqlen_q, seqlen_k, 1.0 / math.sqrt(d) if scale is None else float(scale),
                                int(window_left), **kw)
    return o, lse


def verify_tree(target_probs, draft_probs, tokens, parent, uniform, uniform_next, cu_seqlens_q, most, distinct=False,
                path=None, count=None, next_token=None, workspace=None, **kw):
    """Drafted trees verified (verify_tree_kernel); draft_probs None: the drafts were
    chosen, not drawn; ``distinct``: siblings were drawn without replacement.  Returns
    path [b, most] (the accepted nodes, root first, then -1), count [b] and the
    next token [b].  The workspace (float32) comes from torch's allocator, on the call's
    stream, unless given."""
    b, stream = cu_seqlens_q.shape[0] - 1, kw.get("stream")
    path = _new(tokens, rt.DT_INT32, (b, int(most)), stream) if path is None else path
    count = _new(tokens, rt.DT_INT32, (b,), stream) if count is None else count
    next_token = _new(tokens, 0, (b,), stream) if next_token is None else next_token
    draft = _none(target_probs.dtype, target_probs.device, 2) if draft_probs is None else draft_probs
    if workspace is None:
        workspace = _room(rt.module().verify_tree_workspace(b, tokens.shape[0], target_probs.shape[1]), tokens, stream)
    verify_tree_kernel(target_probs, draft, tokens, parent, uniform, uniform_next, cu_seqlens_q, path, count, next_token,
                       workspace, bool(distinct), **kw)
    return path, count, next_token


def paged_keep_path(k_cache, v_cache, page_table, cu_seqlens_q, seqused_k, path, count, out=None, **kw):
    """Moves the accepted paths' cache rows (paged_keep_path_kernel) and returns the
    keys that each sequence has now [b]."""
    out = _new(seqused_k, 0, seqused_k.shape, kw.get("stream")) if out is None else out
    paged_keep_path_kernel(k_cache, v_cache, page_table, cu_seqlens_q, seqused_k, path, count, out, **kw)
    return out


_GATE_ACTS = {None: 0, "none": 0, "sigmoid": 1, "tanh": 2}


def block_norm(x, h, w_pre, eps, w_post=None, gate=None, gate_act=None, residual_scale=1.0, out=None, norm_out=None,
               **kw):
    """y = residual_scale x + act(gate) norm(h, w_post) and n = norm(y, w_pre)
    (block_norm_kernel); gate broadcasts to x; w_pre None: y only (n is None).
    ``out=x`` and ``norm_out=h`` work in place."""
    import torch
    if gate_act not in _GATE_ACTS:
        raise rt.G950Error(rt.USAGE, f"block_norm: unknown gate_act {gate_act!r}")
    stream = kw.get("stream")
    empty_like = torch.empty_like if stream is None else _on_stream(stream, torch.empty_like)
    y = empty_like(x) if out is None else out
    n = None
    if w_pre is not None:
        n = empty_like(x) if norm_out is None else norm_out
    none = _none(x.dtype, x.device, 1)
    if gate is not None and gate.shape != x.shape:
        gate = gate.expand(x.shape)
    block_norm_kernel(x, h, none if w_post is None else w_post, _none(x.dtype, x.device, 2) if gate is None else gate,
                      none if w_pre is None else w_pre, y, _none(x.dtype, x.device, 2) if n is None else n, float(eps),
                      _GATE_ACTS[gate_act], float(residual_scale), **kw)
    return y, n
