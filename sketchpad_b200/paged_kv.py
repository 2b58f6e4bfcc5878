"""The paged key-value cache of token generation: writing the new tokens and attending to it.

The reference's paged cache for its language models
(crates/sketchpad-core/src/paged_attention.rs, kv_cache.rs) keeps fixed-size blocks of tokens
and a block table per sequence; `PagedKVCache` is that cache on the GPU:

    k, v         [pages, page_size, kv_heads, head_dim], any strides whose last is 1
                 (a [pages, kv_heads, page_size, head_dim] allocation is passed as its
                 transposed view)
    block_table  int32 [sequences, max_pages]: the page of token t is [b, t // page_size];
                 entries outside [0, pages) are pages that are not there

The cache holds bf16 or f16, or e4m3 values times a scale per head.
"""
from __future__ import annotations

from typing import Dict, Optional

import torch

from . import _lib
from ._torch import dtype_code, ptr, require_cuda, stream_ptr


class PagedKVCache:
    """k and v tensors of equal shape; k_scale and v_scale f32 [kv_heads] for e4m3 ones.

    The object keeps the device workspace of `attend`, one per stream that calls it (a call
    captured into a graph that is replayed on another stream needs a `workspace` of its own:
    `new_workspace`)."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                 v_scale: Optional[torch.Tensor] = None):
        self.device = require_cuda(k, v, k_scale, v_scale)
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("k and v must be [pages, page_size, kv_heads, head_dim] alike")
        if k.dtype == torch.float8_e4m3fn:
            self._code = _lib.SP_E4M3
            for s in (k_scale, v_scale):
                if s is None or s.dtype != torch.float32 or s.shape != (k.shape[2],) or \
                        not s.is_contiguous():
                    raise ValueError(f"e4m3 caches need contiguous f32 scales [{k.shape[2]}]")
        elif k.dtype in (torch.bfloat16, torch.float16):
            self._code = dtype_code(k.dtype)
            if k_scale is not None or v_scale is not None:
                raise ValueError("only e4m3 caches have scales")
        else:
            raise TypeError("the cache holds bf16, f16 or float8_e4m3fn")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.pages, self.page_size, self.kv_heads, self.head_dim = k.shape
        self._strides = (_lib.i64_array(k.stride()), _lib.i64_array(v.stride()))
        self._work: Dict[int, torch.Tensor] = {}

    @classmethod
    def allocate(cls, pages: int, page_size: int, kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, device="cuda",
                 k_scale: Optional[torch.Tensor] = None,
                 v_scale: Optional[torch.Tensor] = None) -> "PagedKVCache":
        """A zeroed cache."""
        shape = (pages, page_size, kv_heads, head_dim)
        make = lambda: torch.zeros(shape, dtype=torch.uint8 if dtype == torch.float8_e4m3fn  # noqa: E731
                                   else dtype, device=device).view(dtype)
        return cls(make(), make(), k_scale, v_scale)

    def _table(self, block_table: torch.Tensor) -> torch.Tensor:
        if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.shape[1] == 0:
            raise ValueError("block_table must be int32 [sequences, max_pages]")
        if block_table.stride(1) != 1 or (block_table.stride(0) < block_table.shape[1]
                                          and block_table.shape[0] > 1):
            block_table = block_table.contiguous()
        return block_table

    def append(self, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor,
               seq_ids: torch.Tensor, positions: torch.Tensor, *,
               q: Optional[torch.Tensor] = None, rope: Optional[torch.Tensor] = None,
               q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """Write token i's k[i], v[i] ([tokens, kv_heads, head_dim]) to the slot of position
        positions[i] of sequence seq_ids[i] (int32), and return q[i] ([tokens, heads, head_dim])
        ready for attention.

        rope: f32 [positions, head_dim / 2, 2] (cos, sin) from `rope_pair_table`; k and q are
        rotated by their position (interleaved pairs).  A token whose sequence, position or page
        does not exist (a position of -1, say) is padding: nothing is stored, its q is zeros."""
        dev = require_cuda(k, v, block_table, seq_ids, positions, q, rope, q_out, self.k)
        T = k.shape[0]
        D, hkv = self.head_dim, self.kv_heads
        if k.shape != (T, hkv, D) or v.shape != k.shape or v.dtype != k.dtype:
            raise ValueError(f"k and v must be [tokens, {hkv}, {D}] of one dtype")
        if k.dtype not in (torch.bfloat16, torch.float16) or \
                (self._code != _lib.SP_E4M3 and k.dtype != self.k.dtype):
            raise ValueError("k and v must be of the cache's dtype (bf16 or f16 for e4m3)")
        for t in (seq_ids, positions):
            if t.shape != (T,) or t.dtype != torch.int32 or not t.is_contiguous():
                raise ValueError(f"seq_ids and positions must be contiguous int32 [{T}]")
        table = self._table(block_table)
        hq = 0
        if q is not None:
            hq = q.shape[1] if q.dim() == 3 else 0
            if hq == 0 or q.shape != (T, hq, D) or q.dtype != k.dtype:
                raise ValueError(f"q must be [{T}, heads, {D}] of k's dtype")
            if q_out is None:
                q_out = torch.empty((T, hq, D), dtype=q.dtype, device=dev)
            elif q_out.shape != q.shape or q_out.dtype != q.dtype or not q_out.is_contiguous():
                raise ValueError("q_out must be contiguous and have q's shape and dtype")
            q = _heads(q)
        elif q_out is not None:
            raise ValueError("q_out without q")
        k, v = _heads(k), _heads(v)
        if rope is not None and (rope.dtype != torch.float32 or not rope.is_contiguous()
                                 or rope.dim() != 3 or rope.shape[1:] != (D // 2, 2)):
            raise ValueError(f"rope must be contiguous f32 [positions, {D // 2}, 2]")
        qs = None if q is None else _lib.i64_array((*q.stride(), 0))
        _lib.call("sp_paged_kv_append", ptr(q), ptr(k), ptr(v), ptr(q_out), qs,
                  _lib.i64_array((*k.stride(), 0)), _lib.i64_array((*v.stride(), 0)), T, hq, hkv,
                  D, ptr(self.k), ptr(self.v), ptr(self.k_scale), ptr(self.v_scale),
                  *self._strides, self.pages, self.page_size, ptr(table), table.shape[0],
                  table.shape[1], max(table.stride(0), table.shape[1]), ptr(seq_ids),
                  ptr(positions), ptr(rope), 0 if rope is None else rope.shape[0],
                  dtype_code(k.dtype), self._code, stream_ptr(dev))
        return q_out

    def new_workspace(self, batch: int, heads: int) -> torch.Tensor:
        """A workspace for `attend` calls of up to `batch` sequences and `heads` query heads."""
        n = _lib.load().sp_paged_attention_workspace_size(batch, heads, self.kv_heads)
        return torch.zeros((n + 3) // 4, dtype=torch.int32, device=self.device)

    def attend(self, q: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, *,
               scale: Optional[float] = None, window: Optional[int] = None, sinks: int = 0,
               out: Optional[torch.Tensor] = None,
               workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
        """softmax(scale q k^T) v of one new token per sequence: q [sequences, heads, head_dim]
        over the seq_lens[b] (int32) tokens of sequence b, its own among them; query head h reads
        cache head h // (heads / kv_heads).  window: only the last `window` tokens and the first
        `sinks`.  scale: 1 / sqrt(head_dim) unless given.  A sequence of length 0, or without a
        page that is there, gives zeros."""
        dev = require_cuda(q, block_table, seq_lens, out, workspace, self.k)
        if q.dim() != 3 or q.shape[2] != self.head_dim or q.shape[1] == 0 or \
                q.shape[1] % self.kv_heads:
            raise ValueError(f"q must be [sequences, heads, {self.head_dim}] with heads a "
                             f"multiple of {self.kv_heads}")
        B, hq, D = q.shape
        if q.dtype not in (torch.bfloat16, torch.float16) or \
                (self._code != _lib.SP_E4M3 and q.dtype != self.k.dtype):
            raise ValueError("q must be of the cache's dtype (bf16 or f16 for e4m3)")
        if block_table.shape[0] != B or seq_lens.shape != (B,) or seq_lens.dtype != torch.int32 \
                or not seq_lens.is_contiguous():
            raise ValueError(f"block_table must have {B} rows and seq_lens be contiguous int32 "
                             f"[{B}]")
        if window is not None and window < 1:
            raise ValueError("window must be at least 1")
        if sinks < 0:
            raise ValueError("sinks must not be negative")
        table = self._table(block_table)
        q = _heads(q)
        if out is None:
            out = torch.empty((B, hq, D), dtype=q.dtype, device=dev)
        elif out.shape != (B, hq, D) or out.dtype != q.dtype or not out.is_contiguous():
            raise ValueError(f"out must be contiguous {q.dtype} [{B}, {hq}, {D}]")
        stream = stream_ptr(dev)
        if workspace is None:
            need = _lib.load().sp_paged_attention_workspace_size(B, hq, self.kv_heads)
            workspace = self._work.get(stream.value)
            if workspace is None or workspace.numel() * 4 < need:
                workspace = self._work[stream.value] = self.new_workspace(B, hq)
        elif not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous")
        _lib.call("sp_paged_attention", ptr(q), _lib.i64_array((*q.stride(), 0)), ptr(self.k),
                  ptr(self.v), ptr(self.k_scale), ptr(self.v_scale), *self._strides, ptr(table),
                  table.shape[1], max(table.stride(0), table.shape[1]), ptr(seq_lens), ptr(out),
                  B, hq, self.kv_heads, D, self.pages, self.page_size, window or 0, sinks,
                  float(scale) if scale else 0.0, dtype_code(q.dtype), self._code,
                  ptr(workspace), workspace.numel() * workspace.element_size(), stream)
        return out


def _heads(t: torch.Tensor) -> torch.Tensor:
    """t [tokens, heads, dim] with 16-byte aligned, contiguous heads (else a copy)."""
    if t.stride(2) != 1 or t.stride(0) % 8 or t.stride(1) % 8 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


__all__ = ["PagedKVCache"]
