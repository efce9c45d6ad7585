"""Linears in 8-bit integers with a scale a token and a scale an output channel, on torch device tensors.

    w, w_scales = int8.quantize_rows(weight)               # once: [out_dim, in_dim], a scale a channel
    q, scales = int8.quantize_rows(x, norm=w_norm)         # a step's rows, RMS-normed on the way
    y = int8.matmul(q, scales, w, w_scales)

Each function issues one C-ABI call on the current torch stream of the graph's
device; nothing is read back.
"""
from __future__ import annotations

import torch

from . import capi
from .gguf import GGML_BF16, GGML_F16, GGML_F32
from .ops import RenderGraph
from .serve import _U32, _graph, _vec

_TYPES = {torch.float32: GGML_F32, torch.float16: GGML_F16, torch.bfloat16: GGML_BF16}
_I8 = torch.int8


def _rows(t: torch.Tensor, what: str):
    """(rows, columns, row stride) of a 2-D view with contiguous rows; one row's stride is nothing and counts as a
    whole row of 16-byte pieces."""
    strides = t.stride()
    if len(strides) == 2:
        n, m = t.shape
        row = strides[0] if n > 1 else m + -m % 16
        if (strides[1] == 1 or m <= 1) and 0 <= row <= _U32:
            return n, m, row
    raise ValueError(f"{what} must be a 2-D view with contiguous rows, under 2^32 apart")


def _scales(t: torch.Tensor, what: str, n: int) -> int:
    if t.dtype is not torch.float32 or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous f32 device tensor of {n} elements")
    return t.data_ptr()


def quantize_rows(x: torch.Tensor, norm: torch.Tensor | None = None, eps: float = 1e-6, q: torch.Tensor | None = None,
                  scales: torch.Tensor | None = None, g: RenderGraph | None = None):
    """Rows of x (f32, f16 or bf16 [T, K], K a multiple of 16) -> q int8 [T, K] and scales f32 [T] with scales[t] *
    q[t] standing for x[t], or for its RMS norm with weights norm [K] (llmr_quantize_rows_i8). Returns (q, scales)."""
    T, K, xs = _rows(x, "x")
    t = _TYPES.get(x.dtype)
    if t is None:
        raise ValueError("x must be float32, float16 or bfloat16")
    if q is None:
        q = torch.empty(T, K, dtype=_I8, device=x.device)
    if scales is None:
        scales = torch.empty(T, dtype=torch.float32, device=x.device)
    qn, qk, qs = _rows(q, "q")
    if q.dtype is not _I8 or qn != T or qk != K:
        raise ValueError("q must be int8 with x's shape")
    if norm is not None and norm.numel() != K:
        raise ValueError("norm must have x's columns")
    sp, np_ = _scales(scales, "scales", T), _vec(norm, "norm", K)
    on = (x, q, scales) if norm is None else (x, q, scales, norm)
    _graph(g, *on).ctx.quantize_rows_i8(x.data_ptr(), np_, q.data_ptr(), sp,
                                        capi.QuantizeRowsParams(T, K, t, xs, qs, eps))
    return q, scales


def matmul(x: torch.Tensor, x_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor,
           out: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16,
           g: RenderGraph | None = None) -> torch.Tensor:
    """out[t, n] = x_scales[t] * w_scales[n] * sum_k x[t, k] * w[n, k] (llmr_matmul_i8): x int8 [T, K], w int8 [N, K],
    K a multiple of 16, scales f32 [T] and [N]. out [T, N] f32, f16 or bf16, any N (None: a new one of `dtype`); it
    overlaps no input."""
    M, K, xs = _rows(x, "x")
    N, Kw, ws = _rows(w, "w")
    if x.dtype is not _I8 or w.dtype is not _I8 or Kw != K:
        raise ValueError("x and w must be int8 [rows, in_dim] with the same in_dim")
    if out is None:
        out = torch.empty(M, N, dtype=dtype, device=x.device)
    t = _TYPES.get(out.dtype)
    Mo, No, os_ = _rows(out, "out")
    if t is None or Mo != M or No != N:
        raise ValueError(f"out must be [{M}, {N}] of float32, float16 or bfloat16")
    xp, wp = _scales(x_scales, "x_scales", M), _scales(w_scales, "w_scales", N)
    _graph(g, x, x_scales, w, w_scales, out).ctx.matmul_i8(x.data_ptr(), xp, w.data_ptr(), wp, out.data_ptr(),
                                                           capi.MatmulI8Params(M, N, K, xs, ws, t, os_))
    return out
