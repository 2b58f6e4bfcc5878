"""Root-mean-square norm of a residual stream, in the stream's type or quantized to e4m3.

The pre-norms of the reference's language models (crates/sketchpad-llm), which the denoiser has
no counterpart of.  One pass over the row: the residual is added, the sum kept for the next
layer, and the normalised row written in the input's type (`rms_norm`) or as e4m3 values with
one f32 scale per row (`rms_norm_fp8`), the form that Int4Linear takes.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from ._torch import cuda_index, dtype_code, raw_stream

_norm = _lib.Entry("sp_rms_norm")
_norm_fp8 = _lib.Entry("sp_rms_norm_fp8")


def _like(x: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of x's shape and dtype (empty_like keeps x's strides, and is quicker)."""
    return torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)


def _rows(t: torch.Tensor, n: int):
    """(t, pointer, row stride) of t as rows of n values (a copy only where t has no such view)."""
    if not t.is_contiguous():
        if t.dim() != 2:
            t = t.reshape(-1, n)
        if t.stride(1) != 1 or (t.stride(0) < n and t.shape[0] > 1):
            t = t.clone(memory_format=torch.contiguous_format)
        return t, t.data_ptr(), max(t.stride(0), n)
    return t, t.data_ptr(), n


def _operands(x, weight, residual, residual_out):
    """Checks; (device index, rows, n, x's and the residual's rows, weight's and residual_out's
    pointers, residual_out)."""
    index = cuda_index(x, weight, residual, residual_out)
    shape = x.shape
    n = shape[-1] if shape else 0
    if n == 0:
        raise ValueError("x must have a last dimension of at least one value")
    dtype = x.dtype
    w_ptr = ro_ptr = 0
    if weight is not None:
        if weight.dtype != dtype or weight.shape != (n,) or not weight.is_contiguous():
            raise ValueError(f"weight must be [{n}], contiguous, of x's dtype")
        w_ptr = weight.data_ptr()
    xr = _rows(x, n)
    rr = (None, 0, n)
    if residual is not None:
        if residual.shape != shape or residual.dtype != dtype:
            raise ValueError("residual must have x's shape and dtype")
        rr = _rows(residual, n)
        if residual_out is None:
            residual_out = _like(x)
    if residual_out is not None:
        if residual_out.shape != shape or residual_out.dtype != dtype or \
                not residual_out.is_contiguous():
            raise ValueError("residual_out must be contiguous and have x's shape and dtype")
        ro_ptr = residual_out.data_ptr()
    return index, x.numel() // n, n, xr, rr, w_ptr, ro_ptr, residual_out


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor], eps: float = 1e-6, *,
             residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
             residual_out: Optional[torch.Tensor] = None):
    """r = x + residual (rounded to the dtype); y = r / sqrt(mean(r^2) + eps) * weight.

    Returns y, or (y, r) with a residual.  `out` and `residual_out` receive them; they may be x
    or residual themselves (the stream updated in place)."""
    code = dtype_code(x.dtype)
    index, rows, n, xr, rr, w_ptr, ro_ptr, residual_out = _operands(x, weight, residual,
                                                                    residual_out)
    if out is None:
        out = _like(x)
    elif out.shape != x.shape or out.dtype != x.dtype or not out.is_contiguous():
        raise ValueError("out must be contiguous and have x's shape and dtype")
    else:
        cuda_index(x, out)
        if out.data_ptr() == ro_ptr and rows:
            raise ValueError("out and residual_out must be different memory")
    _norm(xr[1], xr[2], rr[1], rr[2], w_ptr, out.data_ptr(), ro_ptr, rows, n, eps, code,
          raw_stream(index))
    return out if residual is None else (out, residual_out)


def rms_norm_fp8(x: torch.Tensor, weight: Optional[torch.Tensor], eps: float = 1e-6, *,
                 residual: Optional[torch.Tensor] = None,
                 residual_out: Optional[torch.Tensor] = None):
    """rms_norm quantized: (q, scale), or (q, scale, r) with a residual.

    q is float8_e4m3fn of x's shape, scale f32 of its leading dimensions, y = q * scale with
    scale = max|y| / 448 over each row (1 where a row is all zeros)."""
    code = dtype_code(x.dtype)
    index, rows, n, xr, rr, w_ptr, ro_ptr, residual_out = _operands(x, weight, residual,
                                                                    residual_out)
    q = (torch.empty_like(x, dtype=torch.float8_e4m3fn) if x.is_contiguous()
         else x.new_empty(x.shape, dtype=torch.float8_e4m3fn))
    scale = x.new_empty(x.shape[:-1], dtype=torch.float32)
    _norm_fp8(xr[1], xr[2], rr[1], rr[2], w_ptr, q.data_ptr(), scale.data_ptr(), ro_ptr, rows, n,
              eps, code, raw_stream(index))
    return (q, scale) if residual is None else (q, scale, residual_out)


__all__ = ["rms_norm", "rms_norm_fp8"]
