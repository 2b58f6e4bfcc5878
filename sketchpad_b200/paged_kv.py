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

import ctypes
from typing import Dict, Optional

import torch

from . import _lib
from ._torch import (Workspaces, cuda_index, dtype_code, given_workspace, ptr, raw_stream,
                     require_cuda)

_append = _lib.Entry("sp_paged_kv_append")
_attend = _lib.Entry("sp_paged_attention")
_workspaces = Workspaces()
_16BIT = {torch.float16: _lib.SP_F16, torch.bfloat16: _lib.SP_BF16}


class PagedKVCache:
    """k and v tensors of equal shape; k_scale and v_scale f32 [kv_heads] for e4m3 ones.

    The calls of `attend` share one device workspace per stream.  A call that is captured into a
    graph gets one of the graph's, zeroed in every replay, unless it is given one (`new_workspace`),
    which must not be used by work beside the replays."""

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
        self._work_bytes: Dict[int, int] = {}
        self._handle = ctypes.c_void_p()
        _lib.call("sp_paged_cache_create", ptr(k), ptr(v), ptr(k_scale), ptr(v_scale),
                  _lib.i64_array(k.stride()), _lib.i64_array(v.stride()), *k.shape, self._code,
                  ctypes.byref(self._handle))

    def __del__(self):
        try:
            if self._handle:
                _lib.load().sp_paged_cache_destroy(self._handle)
        except Exception:  # pragma: no cover - interpreter shutdown
            pass

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

    @staticmethod
    def _table(block_table: torch.Tensor) -> torch.Tensor:
        if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.shape[1] == 0:
            raise ValueError("block_table must be int32 [sequences, max_pages]")
        if not block_table.is_contiguous():
            s0, s1 = block_table.stride()
            if s1 != 1 or s0 < block_table.shape[1]:
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
        rotated by their position, in interleaved pairs (2 i, 2 i + 1).  (Projections made for
        pairs (i, i + head_dim / 2) have their rows put in that order first: row 2 i + h of a head
        from row i + h head_dim / 2.)  A token whose sequence, position or page
        does not exist (a position of -1, say) is padding: nothing is stored, its q is zeros."""
        index = cuda_index(k, v, block_table, seq_ids, positions, q, rope, q_out, self.k)
        T = k.shape[0]
        D, hkv = self.head_dim, self.kv_heads
        dtype = k.dtype
        if k.shape != (T, hkv, D) or v.shape != k.shape or v.dtype != dtype:
            raise ValueError(f"k and v must be [tokens, {hkv}, {D}] of one dtype")
        code = _16BIT.get(dtype)
        if code is None or (self._code != _lib.SP_E4M3 and code != self._code):
            raise ValueError("k and v must be of the cache's dtype (bf16 or f16 for e4m3)")
        for t in (seq_ids, positions):
            if t.shape != (T,) or t.dtype != torch.int32 or not t.is_contiguous():
                raise ValueError(f"seq_ids and positions must be contiguous int32 [{T}]")
        table = self._table(block_table)
        hq = q_ptr = out_ptr = q_tok = q_head = 0
        if q is not None:
            hq = q.shape[1] if q.dim() == 3 else 0
            if hq == 0 or q.shape != (T, hq, D) or q.dtype != dtype:
                raise ValueError(f"q must be [{T}, heads, {D}] of k's dtype")
            if q_out is None:
                q_out = q.new_empty((T, hq, D))
            elif q_out.shape != q.shape or q_out.dtype != dtype or not q_out.is_contiguous():
                raise ValueError("q_out must be contiguous and have q's shape and dtype")
            q, q_ptr, q_tok, q_head = _heads(q)
            out_ptr = q_out.data_ptr()
        elif q_out is not None:
            raise ValueError("q_out without q")
        k, k_ptr, k_tok, k_head = _heads(k)
        v, v_ptr, v_tok, v_head = _heads(v)
        rope_ptr = rope_rows = 0
        if rope is not None:
            if rope.dtype != torch.float32 or not rope.is_contiguous() or rope.dim() != 3 or \
                    rope.shape[1] != D // 2 or rope.shape[2] != 2:
                raise ValueError(f"rope must be contiguous f32 [positions, {D // 2}, 2]")
            rope_ptr, rope_rows = rope.data_ptr(), rope.shape[0]
        rows, cols = table.shape
        _append(self._handle, q_ptr, k_ptr, v_ptr, out_ptr, q_tok, q_head, k_tok, k_head, v_tok,
                v_head, T, hq, table.data_ptr(), rows, cols, max(table.stride(0), cols),
                seq_ids.data_ptr(), positions.data_ptr(), rope_ptr, rope_rows, code,
                raw_stream(index))
        return q_out

    def workspace_size(self, heads: int) -> int:
        """Bytes of the workspace of an `attend` call of `heads` query heads."""
        return _lib.load().sp_paged_attention_workspace_size(heads, self.kv_heads, self.head_dim)

    def new_workspace(self, heads: int) -> torch.Tensor:
        """A workspace for `attend` calls of `heads` query heads, of any batch."""
        return torch.zeros((self.workspace_size(heads) + 3) // 4, dtype=torch.int32,
                           device=self.device)

    def attend(self, q: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, *,
               scale: Optional[float] = None, window: Optional[int] = None, sinks: int = 0,
               out: Optional[torch.Tensor] = None,
               workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
        """softmax(scale q k^T) v of one new token per sequence: q [sequences, heads, head_dim]
        over the seq_lens[b] (int32) tokens of sequence b, its own among them; query head h reads
        cache head h // (heads / kv_heads).  window: only the last `window` tokens and the first
        `sinks`.  scale: positive, 1 / sqrt(head_dim) unless given.  Lengths beyond the block
        table are cut, tokens on pages that are not there are not seen, and a sequence that sees
        none gives zeros."""
        index = cuda_index(q, block_table, seq_lens, out, workspace, self.k)
        D, hkv = self.head_dim, self.kv_heads
        if q.dim() != 3:
            raise ValueError(f"q must be [sequences, heads, {D}]")
        B, hq, qd = q.shape
        if qd != D or hq == 0 or hq % hkv:
            raise ValueError(f"q must be [sequences, heads, {D}] with heads a multiple of {hkv}")
        code = _16BIT.get(q.dtype)
        if code is None or (self._code != _lib.SP_E4M3 and code != self._code):
            raise ValueError("q must be of the cache's dtype (bf16 or f16 for e4m3)")
        table = self._table(block_table)
        rows, cols = table.shape
        if rows != B or seq_lens.shape != (B,) or seq_lens.dtype != torch.int32 \
                or not seq_lens.is_contiguous():
            raise ValueError(f"block_table must have {B} rows and seq_lens be contiguous int32 "
                             f"[{B}]")
        if window is None:
            window = 0
        elif window < 1:
            raise ValueError("window must be at least 1")
        if sinks < 0:
            raise ValueError("sinks must not be negative")
        if scale is None:
            scale = 0.0  # the entry's own 1 / sqrt(head_dim)
        elif not 2.0 ** -126 <= scale < float("inf"):
            raise ValueError("scale must be positive and finite (None: 1 / sqrt(head_dim))")
        if out is None:
            out = torch.empty_like(q) if q.is_contiguous() else q.new_empty((B, hq, D))
        elif out.shape != (B, hq, D) or out.dtype != q.dtype or not out.is_contiguous():
            raise ValueError(f"out must be contiguous {q.dtype} [{B}, {hq}, {D}]")
        q, q_ptr, q_seq, q_head = _heads(q)
        stream = raw_stream(index)
        if workspace is None:
            need = self._work_bytes.get(hq)
            if need is None:
                need = self._work_bytes[hq] = self.workspace_size(hq)
            work = _workspaces.get(index, stream, need)
        else:
            work = given_workspace(workspace)
        _attend(self._handle, q_ptr, q_seq, q_head, table.data_ptr(), cols,
                max(table.stride(0), cols), seq_lens.data_ptr(), out.data_ptr(), B, hq, window,
                sinks, scale, code, work[1], work[2], stream)
        return out


def _heads(t: torch.Tensor):
    """(t, pointer, token stride, head stride) of t [tokens, heads, dim] with 16-byte aligned,
    contiguous heads, or of a copy that has them."""
    s0, s1, s2 = t.stride()
    p = t.data_ptr()
    if s2 != 1 or s0 % 8 or s1 % 8 or p % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        s0, s1, _ = t.stride()
        p = t.data_ptr()
    return t, p, s0, s1


__all__ = ["PagedKVCache"]
