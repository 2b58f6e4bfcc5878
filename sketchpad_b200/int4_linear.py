"""Linear layers with 4-bit weights and group scales, for few rows of activations.

The weight-only 4-bit linears of a language model that generates a token at a time
(crates/sketchpad-llm runs them as row-wise CPU products, crates/sketchpad-llm/src/quantized.rs
:70-92).  The quantized GEMMs of `GpuQuantizedLinear` work on tiles of 256 rows; here one to a
few dozen rows meet a weight that is streamed once:

    w[n, k] = scale[k // group, n] * (q[n, k] - zero[k // group, n])
    y = x @ w.T (+ bias)

x is bf16, f16, or e4m3 with a scale per row (`rms_norm_fp8`).
"""
from __future__ import annotations

from typing import Optional

import numpy as np
import torch

from . import _lib
from ._torch import (Workspaces, cuda_index, dtype_code, given_workspace, ptr, raw_stream,
                     require_cuda, stream_ptr)

_linear = _lib.Entry("sp_int4_linear")
_workspaces = Workspaces()

_X = {torch.float16: _lib.SP_F16, torch.bfloat16: _lib.SP_BF16,
      torch.float8_e4m3fn: _lib.SP_E4M3}


class Int4Linear:
    """qweight uint8 [N, K/2] (even k in the low nibble), scales f16 / bf16 [K/group, N], zeros
    uint8 [K/group, N] with values 0..15 (None: 8, symmetric weights), bias [N].

    group_size: 32, 64 or a multiple of 128 that divides K.  The constructor lays the weight out
    for the kernels once, and the bias in each output type (device copies; the given tensors are
    not kept, and changing them later changes no output)."""

    def __init__(self, qweight: torch.Tensor, scales: torch.Tensor,
                 zeros: Optional[torch.Tensor] = None, *, group_size: int,
                 bias: Optional[torch.Tensor] = None):
        dev = require_cuda(qweight, scales, zeros, bias)
        if qweight.dim() != 2 or qweight.dtype != torch.uint8:
            raise ValueError("qweight must be uint8 [out_features, in_features / 2]")
        N, K = qweight.shape[0], 2 * qweight.shape[1]
        sizes = _lib.i64_array((0, 0, 0, 0))
        _lib.call("sp_int4_packed_bytes", N, K, group_size, sizes)
        if scales.dtype not in (torch.float16, torch.bfloat16) or \
                scales.shape != (K // group_size, N):
            raise ValueError(f"scales must be f16 or bf16 [{K // group_size}, {N}]")
        if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != scales.shape):
            raise ValueError("zeros must be uint8 of the scales' shape")
        if bias is not None and bias.shape != (N,):
            raise ValueError(f"bias must be [{N}]")
        qweight, scales = qweight.contiguous(), scales.contiguous()
        zeros = None if zeros is None else zeros.contiguous()
        self.out_features, self.in_features, self.group_size = N, K, group_size
        self.scale_dtype = scales.dtype
        self.bias = None if bias is None else bias.detach().clone()
        self._bias = {} if bias is None else {
            dt: self.bias.to(dt).contiguous()
            for dt in (torch.float32, torch.float16, torch.bfloat16)}
        self._work_bytes = {}
        self.q = torch.empty(sizes[0], dtype=torch.uint8, device=dev)
        self.scale = torch.empty(sizes[1], dtype=torch.uint8, device=dev)
        self.zero = None if zeros is None else torch.empty(sizes[2], dtype=torch.uint8, device=dev)
        _lib.call("sp_int4_repack", ptr(qweight), ptr(scales), ptr(zeros), N, K, group_size,
                  ptr(self.q), ptr(self.scale), ptr(self.zero), stream_ptr(dev))
        self._weight_args = (self.q.data_ptr(), self.scale.data_ptr(),
                             0 if zeros is None else self.zero.data_ptr(),
                             dtype_code(scales.dtype))

    @classmethod
    def from_weight(cls, weight: torch.Tensor, group_size: int = 128, symmetric: bool = True,
                    scale_dtype: torch.dtype = torch.float16,
                    bias: Optional[torch.Tensor] = None) -> "Int4Linear":
        """Quantize a float weight [N, K] by rounding to nearest: symmetric groups take scale =
        max|w| / 7 (values -8..7 around 8), others the range [min, max] with 0 in it."""
        N, K = weight.shape
        if K % group_size:
            raise ValueError(f"{K} inputs are not a multiple of the group of {group_size}")
        w = weight.float().reshape(N, K // group_size, group_size)
        if symmetric:
            s = (w.abs().amax(-1) / 7).to(scale_dtype)
            z = torch.full_like(s, 8.0, dtype=torch.float32)
        else:
            lo, hi = w.amin(-1).clamp(max=0), w.amax(-1).clamp(min=0)
            s = ((hi - lo) / 15).to(scale_dtype)
            z = torch.round(-lo / torch.where(s == 0, 1, s.float())).clamp(0, 15)
        sf = torch.where(s == 0, 1, s.float())
        q = (torch.round(w / sf[..., None]) + z[..., None]).clamp(0, 15).to(torch.uint8)
        q = q.reshape(N, K)
        packed = q[:, 0::2] | (q[:, 1::2] << 4)
        zeros = None if symmetric else z.to(torch.uint8).t().contiguous()
        return cls(packed, s.t().contiguous(), zeros, group_size=group_size, bias=bias)

    @classmethod
    def from_gguf_q4_0(cls, data, out_features: int, in_features: int, device="cuda",
                       bias: Optional[torch.Tensor] = None) -> "Int4Linear":
        """GGUF Q4_0 bytes (per 32 values an f16 scale and 16 bytes: value i in the low nibble of
        byte i, value 16 + i in the high one; value = scale * (q - 8)), losslessly."""
        buf = np.frombuffer(bytes(data), np.uint8) if not isinstance(data, np.ndarray) else data
        if in_features % 32 or buf.size != out_features * (in_features // 32) * 18:
            raise ValueError("Q4_0 rows are blocks of 18 bytes per 32 values")
        blocks = torch.from_numpy(np.array(buf).reshape(out_features, in_features // 32, 18))
        scales = blocks[..., :2].contiguous().view(torch.float16)[..., 0].t().contiguous()
        b = blocks[..., 2:]
        q = torch.cat((b & 15, b >> 4), -1).reshape(out_features, in_features)
        packed = q[:, 0::2] | (q[:, 1::2] << 4)
        return cls(packed.to(device), scales.to(device), None, group_size=32, bias=bias)

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The weight's values [N, K]; f32 is scale * (q - zero) exactly."""
        out = torch.empty((self.out_features, self.in_features), dtype=dtype,
                          device=self.q.device)
        q, s, z, sd = self._weight_args
        _lib.call("sp_int4_dequant", q, s, z, self.out_features, self.in_features,
                  self.group_size, sd, ptr(out), dtype_code(dtype), stream_ptr(self.q.device))
        return out

    def forward(self, x: torch.Tensor, x_scale: Optional[torch.Tensor] = None, *,
                out_dtype: Optional[torch.dtype] = None,
                out: Optional[torch.Tensor] = None,
                workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
        """[..., in_features] -> [..., out_features].

        x bf16 or f16, or float8_e4m3fn with x_scale f32 [...].  The output's type is
        out_dtype, else out's, else x's (bf16 for e4m3).

        The layers share one workspace per stream.  A call that is captured into a graph gets one
        of the graph's, zeroed in every replay, unless it is given one (`workspace_size` zero
        bytes), which must not be used by work beside the replays."""
        index = cuda_index(x, self.q, x_scale, out, workspace)
        N, K = self.out_features, self.in_features
        xd = _X.get(x.dtype)
        if xd is None:
            raise TypeError("x must be bf16, f16 or float8_e4m3fn")
        shape = x.shape
        if not shape or shape[-1] != K:
            raise ValueError(f"x must be [..., {K}]")
        s_ptr = 0
        if xd == _lib.SP_E4M3:
            if x_scale is None:
                raise ValueError("e4m3 activations come with x_scale")
            if x_scale.shape != shape[:-1] or x_scale.dtype != torch.float32 or \
                    not x_scale.is_contiguous():
                raise ValueError(f"x_scale must be contiguous f32 {tuple(shape[:-1])}")
            s_ptr, align = x_scale.data_ptr(), 8
        elif x_scale is not None:
            raise ValueError("only e4m3 activations come with x_scale")
        else:
            align = 16
        dt = out_dtype or (out.dtype if out is not None else
                           torch.bfloat16 if xd == _lib.SP_E4M3 else x.dtype)
        if out is None:
            out = x.new_empty((*shape[:-1], N), dtype=dt)
        elif out.dtype != dt or out.shape != (*shape[:-1], N) or not out.is_contiguous():
            raise ValueError(f"out must be contiguous {dt} [..., {N}]")
        M, stride, p = x.numel() // K, K, x.data_ptr()
        if p % align or not x.is_contiguous():
            x = x if x.dim() == 2 else x.reshape(-1, K)
            stride, p = x.stride(0), x.data_ptr()
            if x.stride(1) != 1 or p % align or (M > 1 and (stride % 8 or stride < K)):
                x = x.clone(memory_format=torch.contiguous_format)
                p, stride = x.data_ptr(), K
            elif M <= 1:
                stride = K
        code = dtype_code(dt)
        b_ptr = self._bias[dt].data_ptr() if self._bias else 0
        raw = raw_stream(index)
        if workspace is None:
            tile = 8 if M <= 8 else 16 if M <= 16 else 32
            need = self._work_bytes.get(tile)
            if need is None:
                need = self._work_bytes[tile] = self.workspace_size(tile)
            work = _workspaces.get(index, raw, need)
        else:
            work = given_workspace(workspace)
        _linear(p, stride, xd, s_ptr, *self._weight_args, b_ptr, out.data_ptr(), M, N, K,
                self.group_size, code, work[1], work[2], raw)
        return out

    def workspace_size(self, rows: int) -> int:
        """Bytes of a workspace (zeros, any dtype) for a call of that many rows."""
        return _lib.load().sp_int4_linear_workspace_size(rows, self.out_features,
                                                         self.in_features, self.group_size)

    __call__ = forward


__all__ = ["Int4Linear"]
