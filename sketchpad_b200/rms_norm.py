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
from ._torch import dtype_code, ptr, require_cuda, stream_ptr


def _rows(t: torch.Tensor, n: int) -> torch.Tensor:
    """t as rows of n values with one row stride (a copy only where t has no such view)."""
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= n:
        return t
    t = t.reshape(-1, n)
    return t if t.stride(1) == 1 and (t.stride(0) >= n or t.shape[0] == 1) else t.contiguous()


def _operands(x, weight, residual, residual_out):
    dev = require_cuda(x, weight, residual, residual_out)
    code = dtype_code(x.dtype)
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError("x must have a last dimension of at least one value")
    n = x.shape[-1]
    if weight is not None and (weight.dtype != x.dtype or weight.shape != (n,)
                               or weight.stride(0) != 1):
        raise ValueError(f"weight must be [{n}], contiguous, of x's dtype")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError("residual must have x's shape and dtype")
    if residual_out is not None and (
            residual_out.shape != x.shape or residual_out.dtype != x.dtype
            or not residual_out.is_contiguous()):
        raise ValueError("residual_out must be contiguous and have x's shape and dtype")
    return dev, code, n


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor], eps: float = 1e-6, *,
             residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
             residual_out: Optional[torch.Tensor] = None):
    """r = x + residual (rounded to the dtype); y = r / sqrt(mean(r^2) + eps) * weight.

    Returns y, or (y, r) with a residual.  `out` and `residual_out` receive them; they may be x
    or residual themselves (the stream updated in place)."""
    dev, code, n = _operands(x, weight, residual, residual_out)
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=dev)
    elif out.shape != x.shape or out.dtype != x.dtype or not out.is_contiguous():
        raise ValueError("out must be contiguous and have x's shape and dtype")
    else:
        require_cuda(x, out)
    if residual is not None and residual_out is None:
        residual_out = torch.empty(x.shape, dtype=x.dtype, device=dev)
    xr = _rows(x, n)
    rr = None if residual is None else _rows(residual, n)
    _lib.call("sp_rms_norm", ptr(xr), max(xr.stride(0), n), ptr(rr),
              n if rr is None else max(rr.stride(0), n), ptr(weight), ptr(out), ptr(residual_out),
              xr.shape[0], n, eps, code, stream_ptr(dev))
    return out if residual is None else (out, residual_out)


def rms_norm_fp8(x: torch.Tensor, weight: Optional[torch.Tensor], eps: float = 1e-6, *,
                 residual: Optional[torch.Tensor] = None,
                 residual_out: Optional[torch.Tensor] = None):
    """rms_norm quantized: (q, scale), or (q, scale, r) with a residual.

    q is float8_e4m3fn of x's shape, scale f32 of its leading dimensions, y = q * scale with
    scale = max|y| / 448 over each row (1 where a row is all zeros)."""
    dev, code, n = _operands(x, weight, residual, residual_out)
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=dev)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev)
    if residual is not None and residual_out is None:
        residual_out = torch.empty(x.shape, dtype=x.dtype, device=dev)
    xr = _rows(x, n)
    rr = None if residual is None else _rows(residual, n)
    _lib.call("sp_rms_norm_fp8", ptr(xr), max(xr.stride(0), n), ptr(rr),
              n if rr is None else max(rr.stride(0), n), ptr(weight), ptr(q), ptr(scale),
              ptr(residual_out), xr.shape[0], n, eps, code, stream_ptr(dev))
    return (q, scale) if residual is None else (q, scale, residual_out)


__all__ = ["rms_norm", "rms_norm_fp8"]
