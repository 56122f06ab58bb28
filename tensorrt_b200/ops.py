"""torch-tensor front end of the C ABI (include/bert_b200.h).

torch is used only to own device memory and streams; every function forwards raw pointers to
libbert_b200.so. Names follow the reference free functions they replace
(embSkipLayerNorm, computeSkipLayerNorm, computeMaskIdx, convertMask, MHARunner::run, FC enqueue).
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from . import _lib
from ._lib import check, lib

FP32, FP16, INT8 = 0, 1, 2
ACT_NONE, ACT_GELU_ERF = 0, 1

_TYPE_ID = {torch.float32: FP32, torch.float16: FP16, torch.int8: INT8}


def _ptr(t: torch.Tensor | None):
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("tensorrt_b200 kernels need CUDA tensors; there is no CPU path")
    if not t.is_contiguous():
        raise ValueError("tensor must be contiguous")
    return t.data_ptr()  # ctypes takes the number; an object around every pointer was a quarter of a call's host time


def _stream():
    # A call on a few rows takes the GPU less time than the host: is_available() and a Stream object only before the first use.
    if torch.cuda.is_initialized():
        return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())
    if not torch.cuda.is_available():
        raise ValueError("tensorrt_b200 kernels need a CUDA device; there is no CPU path")
    return torch.cuda.current_stream().cuda_stream


def skip_layer_norm(x, skip, gamma, beta, bias=None, out=None):
    """FP32/FP16 residual + bias + LayerNorm over the last dimension."""
    ld = x.shape[-1]
    out = torch.empty_like(x) if out is None else out
    check(lib.bert_b200_skip_layer_norm(_stream(), _TYPE_ID[x.dtype], ld, x.numel(), _ptr(x), _ptr(skip), _ptr(beta),
                                        _ptr(gamma), _ptr(out), _ptr(bias)), "skip_layer_norm")
    return out


def skip_layer_norm_dqq(x, skip, gamma, beta, bias, dq_in, dq_skip, q_scale, out=None):
    """INT8 in/out residual + bias + LayerNorm (linear layout); gamma/beta/bias FP16."""
    ld = x.shape[-1]
    out = torch.empty_like(x) if out is None else out
    check(lib.bert_b200_skip_layer_norm_dqq(_stream(), ld, x.numel(), _ptr(x), _ptr(skip), _ptr(beta), _ptr(gamma),
                                            _ptr(out), _ptr(bias), dq_in, dq_skip, q_scale), "skip_layer_norm_dqq")
    return out


def skip_layer_norm_interleaved(x, skip, gamma, beta, dq_in, dq_skip, q_scale, q_skip_scale=None):
    """INT8 CHW32 [ld/32, total, 32]; returns out, or (out, preln) when q_skip_scale is given (MTron)."""
    g, total, _ = x.shape
    ld = g * 32
    out = torch.empty_like(x)
    if q_skip_scale is None:
        check(lib.bert_b200_skip_layer_norm_interleaved_hface(_stream(), ld, total, _ptr(x), _ptr(skip), _ptr(beta),
                                                              _ptr(gamma), _ptr(out), dq_in, dq_skip, q_scale),
              "skip_layer_norm_interleaved_hface")
        return out
    preln = torch.empty_like(x)
    check(lib.bert_b200_skip_layer_norm_interleaved_mtron(_stream(), ld, total, _ptr(x), _ptr(skip), _ptr(beta),
                                                          _ptr(gamma), _ptr(out), _ptr(preln), dq_in, dq_skip, q_scale,
                                                          q_skip_scale), "skip_layer_norm_interleaved_mtron")
    return out, preln


def emb_layer_norm(input_ids, token_ids, word_emb, pos_emb, tok_emb, gamma, beta, q_scale=None, mask=None):
    """Fixed layout: ids [S, B] int32 -> [S, B, E]; optional fused INT8 copy when q_scale is given; with the [S, B] int32
    `mask` the same launch also returns the mask index [B] (last element of the result)."""
    S, B = input_ids.shape
    ld = word_emb.shape[1]
    out = torch.empty((S, B, ld), dtype=word_emb.dtype, device=word_emb.device)
    out_i8 = torch.empty((S, B, ld), dtype=torch.int8, device=word_emb.device) if q_scale is not None else None
    mask_idx = torch.empty((B,), dtype=torch.int32, device=word_emb.device) if mask is not None else None
    if mask is not None and (tuple(mask.shape) != (S, B) or mask.dtype != torch.int32 or not mask.is_contiguous()):
        raise ValueError("mask must be a contiguous int32 [S, B] tensor")
    check(lib.bert_b200_emb_layer_norm_mask_idx(_stream(), _TYPE_ID[word_emb.dtype], ld, B, S, _ptr(input_ids),
                                                _ptr(token_ids), _ptr(beta), _ptr(gamma), _ptr(word_emb), _ptr(pos_emb),
                                                _ptr(tok_emb), word_emb.shape[0], tok_emb.shape[0], pos_emb.shape[0],
                                                _ptr(out), _ptr(out_i8), q_scale or 0.0, _ptr(mask), _ptr(mask_idx)),
          "emb_layer_norm")
    res = [out]
    if q_scale is not None:
        res.append(out_i8)
    if mask is not None:
        res.append(mask_idx)
    return res[0] if len(res) == 1 else tuple(res)


def emb_layer_norm_var_seqlen(input_ids, token_ids, cu_seqlens, max_seqlen, word_emb, pos_emb, tok_emb, gamma, beta,
                              with_skip=False, q_scale=None):
    """Packed layout: ids [total] -> [total, E] (+ pre-LN sum when with_skip, + INT8 copy when q_scale)."""
    total = input_ids.shape[0]
    B = cu_seqlens.shape[0] - 1
    ld = word_emb.shape[1]
    out = torch.empty((total, ld), dtype=word_emb.dtype, device=word_emb.device)
    skip = torch.empty_like(out) if with_skip else None
    out_i8 = torch.empty((total, ld), dtype=torch.int8, device=word_emb.device) if q_scale is not None else None
    check(lib.bert_b200_emb_layer_norm_var_seqlen(_stream(), _TYPE_ID[word_emb.dtype], ld, B, max_seqlen, total,
                                                  _ptr(input_ids), _ptr(token_ids), _ptr(cu_seqlens), _ptr(beta),
                                                  _ptr(gamma), _ptr(word_emb), _ptr(pos_emb), _ptr(tok_emb),
                                                  word_emb.shape[0], tok_emb.shape[0], pos_emb.shape[0], _ptr(out), _ptr(skip),
                                                  _ptr(out_i8), q_scale or 0.0), "emb_layer_norm_var_seqlen")
    res = [out]
    if with_skip:
        res.append(skip)
    if q_scale is not None:
        res.append(out_i8)
    return res[0] if len(res) == 1 else tuple(res)


def compute_mask_idx(mask_sb):
    S, B = mask_sb.shape
    out = torch.empty((B,), dtype=torch.int32, device=mask_sb.device)
    check(lib.bert_b200_compute_mask_idx(_stream(), S, B, _ptr(mask_sb), _ptr(out)), "compute_mask_idx")
    return out


def convert_mask(mask_sb, warps_m, warps_n, warps_k=1):
    S, B = mask_sb.shape
    xm = (S + 16 * warps_m - 1) // (16 * warps_m)
    out = torch.empty((B, xm, warps_m * warps_n * warps_k * 32), dtype=torch.int32, device=mask_sb.device)
    check(lib.bert_b200_convert_mask(S, B, warps_m, warps_n, warps_k, _ptr(mask_sb), _ptr(out), _stream()),
          "convert_mask")
    return out


def packed_mask_to_lengths(packed, S, warps_m, warps_n):
    """packed: [B, words] int32/uint32 as written by convert_mask -> lengths [B] int32."""
    B = packed.shape[0]
    row_words = packed[0].numel()
    out = torch.empty((B,), dtype=torch.int32, device=packed.device)
    check(lib.bert_b200_packed_mask_to_lengths(_stream(), S, B, warps_m, warps_n, row_words, _ptr(packed), _ptr(out)),
          "packed_mask_to_lengths")
    return out


def lengths_to_cu_seqlens(lengths):
    B = lengths.shape[0]
    out = torch.empty((B + 1,), dtype=torch.int32, device=lengths.device)
    check(lib.bert_b200_lengths_to_cu_seqlens(_stream(), B, _ptr(lengths), _ptr(out)), "lengths_to_cu_seqlens")
    return out


def fc(a, wt, bias=None, activation=ACT_NONE, alpha=1.0, out_dtype=None, out_scale=1.0, status=None, out=None):
    """C[m, n] = epilogue(A[m, k] . Wt[n, k]); Wt is the [n, k] (transposed) weight."""
    m, k = a.shape
    n = wt.shape[0]
    out_dtype = a.dtype if out_dtype is None else out_dtype
    out = torch.empty((m, n), dtype=out_dtype, device=a.device) if out is None else out
    p = _lib.FcParams(_TYPE_ID[a.dtype], _TYPE_ID[out_dtype], m, n, k, _ptr(a), a.stride(0), _ptr(wt), _ptr(out),
                      out.stride(0), _ptr(bias), activation, alpha, out_scale, _ptr(status))
    check(lib.bert_b200_fc(C.byref(p), _stream()), "fc")
    return out


def _here(*tensors):
    """The operators below run on the current device and its current stream; tensors of another device are refused."""
    dev = torch._C._cuda_getDevice() if torch.cuda.is_initialized() else None
    for t in tensors:
        if t is not None and t.get_device() != dev:
            if not t.is_cuda:
                raise ValueError("tensorrt_b200 kernels need CUDA tensors; there is no CPU path")
            raise ValueError(f"tensor on {t.device}, which is not the current device")


def _vector(t, n, what):
    """Pointer of a contiguous FP32 vector of n values."""
    if t.dtype is not torch.float32 or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous float32 vector of {n} values, got {t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


def _row_stride(t, what, multiple=1):
    """Row stride of a matrix whose rows are contiguous (views of wider tensors are fine)."""
    (rows, width), (stride, step) = t.shape, t.stride()
    if step != 1 and width > 1:
        raise ValueError(f"{what}: the values of a row must be contiguous")
    return stride if rows > 1 else -(-width // multiple) * multiple  # of a single row the stride says nothing


def quantize_rows(x):
    """FP16/FP32 [..., width] -> (INT8 of the same shape, FP32 scale of each row): scale = max|row| / 127, values rounded to nearest even.
    A matrix may be a view with a row stride. The INT8 rows begin on 16 bytes, so they are a view where the width is not a multiple of
    16. Also makes per-channel weights for fc_rowwise out of an [n, k] weight. A row of zeros has scale 0, a row with NaN or infinity
    scale NaN."""
    _here(x)
    if x.dim() != 2:
        if x.dim() == 0 or not x.is_contiguous():
            raise ValueError("quantize_rows: a tensor that is no matrix must be contiguous, with at least one dimension")
        q, scales = quantize_rows(x.view(-1, x.shape[-1]))
        return q.unflatten(0, x.shape[:-1]) if x.dim() > 2 else q[0], scales.view(x.shape[:-1])
    if x.dtype is not torch.float16 and x.dtype is not torch.float32:
        raise ValueError(f"quantize_rows takes float16 or float32, not {x.dtype}")
    rows, width = x.shape
    stride = (width + 15) & ~15
    q = x.new_empty((rows, stride), dtype=torch.int8)
    scales = x.new_empty(rows, dtype=torch.float32)
    check(lib.bert_b200_quantize_rows(_stream(), _TYPE_ID[x.dtype], rows, width, x.data_ptr(), _row_stride(x, "quantize_rows"), q.data_ptr(), stride,
                                      scales.data_ptr()), "quantize_rows")
    return (q if stride == width else q[:, :width]), scales


def fc_rowwise(a, a_scales, wt, wt_scales, bias=None, activation=ACT_NONE, out_dtype=torch.float16, status=None, out=None):
    """C[m, n] = act((A[m, k] . Wt[n, k]) * a_scales[m] * wt_scales[n] + bias[n]): INT8 operands as quantize_rows gives them, FP16 or FP32
    result, any sizes. Rows of A, Wt and `out` begin on 16 bytes (they may be views of wider tensors); without `out`, a result whose rows would
    not is a view of padded rows."""
    _here(a, a_scales, wt, wt_scales, bias, status, out)
    if a.dtype is not torch.int8 or wt.dtype is not torch.int8 or a.dim() != 2 or wt.dim() != 2 or a.shape[1] != wt.shape[1]:
        raise ValueError(f"fc_rowwise takes int8 matrices [m, k] and [n, k], got {a.dtype} {tuple(a.shape)} and {wt.dtype} {tuple(wt.shape)}")
    if out_dtype is not torch.float16 and out_dtype is not torch.float32:
        raise ValueError(f"fc_rowwise gives float16 or float32, not {out_dtype}")
    m, k = a.shape
    n = wt.shape[0]
    per = 8 if out_dtype is torch.float16 else 4
    if out is None:
        if n % per == 0:
            out = a.new_empty((m, n), dtype=out_dtype)
            ldc = n
        else:  # whole lines of 128 bytes: 640 x 30522 FP32 44 us with rows padded to 16 bytes, 37 us so
            ldc = -(-n // (8 * per)) * 8 * per
            out = a.new_empty((m, ldc), dtype=out_dtype)[:, :n]
    elif out.dtype is not out_dtype or out.shape != (m, n):
        raise ValueError(f"out must be a {out_dtype} tensor of shape {(m, n)}")
    else:
        ldc = _row_stride(out, "out", per)
    p = _lib.FcRowwiseParams(_TYPE_ID[out_dtype], activation, m, n, k, a.data_ptr(), _row_stride(a, "a", 16), _vector(a_scales, m, "a_scales"),
                             wt.data_ptr(), _row_stride(wt, "wt", 16), _vector(wt_scales, n, "wt_scales"), out.data_ptr(), ldc,
                             None if bias is None else _vector(bias, n, "bias"), _ptr(status))
    check(lib.bert_b200_fc_rowwise(C.byref(p), _stream()), "fc_rowwise")
    return out


def skip_layer_norm_quantize(x, skip, gamma, beta, bias=None, eps=0.0, with_output=True):
    """Residual (+ bias) + LayerNorm over the last dimension whose result is also quantised row by row: (y, INT8 rows, FP32 scales). `skip` None:
    LayerNorm alone; with_output False: y is None. y has the bits of skip_layer_norm (whose FP16 form has eps 0); the INT8 rows are those
    of the FP32 result before it is rounded to y's type. They feed fc_rowwise where the width is a multiple of 16."""
    _here(x, skip, gamma, beta, bias)
    shape, dtype = x.shape, x.dtype
    if (dtype is not torch.float16 and dtype is not torch.float32) or not shape:
        raise ValueError(f"skip_layer_norm_quantize takes float16 or float32 rows, got {dtype} {tuple(shape)}")
    ld = shape[-1]
    if skip is not None and (skip.dtype is not dtype or skip.shape != shape):
        raise ValueError(f"skip_layer_norm_quantize: skip must be {dtype} of shape {tuple(shape)}, got {skip.dtype} {tuple(skip.shape)}")
    for t in (gamma, beta) if bias is None else (gamma, beta, bias):
        if t.dtype is not dtype or t.shape != (ld,):
            raise ValueError(f"skip_layer_norm_quantize: gamma, beta and bias must be {dtype} of shape {(ld,)}, got {t.dtype} {tuple(t.shape)}")
    x_ptr = _ptr(x)
    y = torch.empty_like(x) if with_output else None
    q = torch.empty_like(x, dtype=torch.int8)
    scales = x.new_empty(shape[:-1], dtype=torch.float32)
    check(lib.bert_b200_skip_layer_norm_quantize(_stream(), _TYPE_ID[dtype], ld, x.numel(), x_ptr, _ptr(skip), _ptr(beta), _ptr(gamma),
                                                 None if y is None else y.data_ptr(), q.data_ptr(), scales.data_ptr(), _ptr(bias), eps),
          "skip_layer_norm_quantize")
    return y, q, scales


class LogProbs(NamedTuple):
    log_probs: torch.Tensor | None       # [rows, tokens]
    entropy: torch.Tensor                # [rows]
    top_ids: torch.Tensor | None         # [rows, top_k]
    top_log_probs: torch.Tensor | None


def token_log_probs(logits, token_ids=None, top_k=0, status=None):
    """Log probabilities of given tokens, entropy and the top_k (at most 32) most likely tokens of each row of FP16/FP32 logits [rows, vocab], a
    matrix or a view with a row stride. token_ids: int32 [rows, tokens] or [rows]; ids outside the vocabulary have probability 0. Tokens of
    logit -inf are no alternatives (ids -1 where too few are left); rows with NaN or +inf give NaN. Masks of the type's lowest value are
    right but slow where they leave less than top_k tokens of a long stretch of the vocabulary (it is read twice): mask with -inf."""
    _here(logits, token_ids, status)
    if (logits.dtype is not torch.float16 and logits.dtype is not torch.float32) or logits.dim() != 2:
        raise ValueError(f"token_log_probs takes float16 or float32 logits [rows, vocab], got {logits.dtype} {tuple(logits.shape)}")
    rows, vocab = logits.shape
    tokens, lp, ids, top = 0, None, None, None
    if token_ids is not None:
        if token_ids.dtype is not torch.int32 or token_ids.dim() not in (1, 2) or token_ids.shape[0] != rows or not token_ids.is_contiguous():
            raise ValueError(f"token_ids must be a contiguous int32 tensor [{rows}, tokens] or [{rows}], got {token_ids.dtype} {tuple(token_ids.shape)}")
        tokens = token_ids.shape[1] if token_ids.dim() == 2 else 1
        lp = torch.empty_like(token_ids, dtype=torch.float32)
    entropy = logits.new_empty(rows, dtype=torch.float32)
    if top_k > 0:
        ids = logits.new_empty((rows, top_k), dtype=torch.int32)
        top = torch.empty_like(ids, dtype=torch.float32)
    p = _lib.LogProbsParams(_TYPE_ID[logits.dtype], rows, vocab, logits.data_ptr(), _row_stride(logits, "token_log_probs"), tokens,
                            token_ids.data_ptr() if tokens else None, top_k, lp.data_ptr() if tokens else None, entropy.data_ptr(),
                            None if ids is None else ids.data_ptr(), None if top is None else top.data_ptr(), _ptr(status))
    check(lib.bert_b200_token_log_probs(C.byref(p), _stream()), "token_log_probs")
    return LogProbs(lp, entropy, ids, top)


def attention_bnsd(q, k, v, kv_lengths=None, scale_bmm1=None, scale_softmax=1.0, scale_bmm2=1.0, status=None):
    """Fused attention on separate q, k, v of shape [B, N, S, d]; returns [B, N, S, d]."""
    B, N, S, d = q.shape
    out = torch.empty_like(q)
    if scale_bmm1 is None:
        scale_bmm1 = d ** -0.5
    p = _lib.AttentionBnsdParams(_TYPE_ID[q.dtype], B, S, N, d, _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(kv_lengths),
                                 scale_bmm1, scale_softmax, scale_bmm2, _ptr(status))
    check(lib.bert_b200_attention_bnsd(C.byref(p), _stream()), "attention_bnsd")
    return out


def mha(qkv, B, S, num_heads, head_size=64, cu_seqlens=None, mask_idx=None, scale_bmm1=None, scale_softmax=1.0,
        scale_bmm2=1.0, status=None, interleaved=False, workspace=None, use_workspace=True, out=None):
    """Fused attention. qkv: fixed [S, B, 3*N*d] (cu_seqlens None), packed [total, 3*N*d], or with
    interleaved=True the INT8 CHW32 form [3*N*d/32, total, 32] (output [N*d/32, total, 32]). `out`: a tensor of the
    output's shape and type to write into instead of a new one. No kernel needs a workspace: `use_workspace` changes nothing."""
    E = num_heads * head_size
    if interleaved:
        total = qkv.shape[1]
        shape = (E // 32, total, 32)
    elif cu_seqlens is None:
        shape = (S, B, E)
        total = 0
    else:
        total = qkv.shape[0]
        shape = (total, E)
    if out is None:
        out = torch.empty(shape, dtype=qkv.dtype, device=qkv.device)
    elif tuple(out.shape) != shape or out.dtype != qkv.dtype or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {qkv.dtype} tensor of shape {shape}")
    if scale_bmm1 is None:
        scale_bmm1 = head_size ** -0.5
    p = _lib.MhaParams(_TYPE_ID[qkv.dtype], B, S, num_heads, head_size, total, _ptr(qkv), _ptr(out), _ptr(cu_seqlens),
                       _ptr(mask_idx), 1 if interleaved else 0, scale_bmm1, scale_softmax, scale_bmm2, _ptr(status))
    if workspace is not None:  # no kernel needs one (bert_b200_mha_workspace_size is 0): nothing is asked for or allocated
        p.workspace, p.workspace_bytes = _ptr(workspace), workspace.numel() * workspace.element_size()
    check(lib.bert_b200_mha(C.byref(p), _stream()), "mha")
    return out
