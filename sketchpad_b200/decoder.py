"""A decoder that generates a token at a time over a paged cache: the token operators together.

The pre-norm decoder layers of the reference's language models (crates/sketchpad-llm): RMS norm,
attention with rotary embedding and grouped key / value heads, SwiGLU feed-forward, 4-bit
weights.  One `step` takes the hidden states of one new token per sequence through every layer:

    rms_norm_fp8 -> qkv (4 bits) -> append to the cache (RoPE) -> attend -> out projection
    rms_norm_fp8 (residual added) -> gate and up (4 bits) -> SwiGLU -> down

Nothing in a step depends on the host (lengths and block tables are device tensors), so a step
can be captured into a CUDA graph once and replayed for every token.

    python -m sketchpad_b200.decoder        # a small random model, tokens per second
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import List, NamedTuple, Optional

import torch

from .glu import swiglu
from .int4_linear import Int4Linear
from .paged_kv import PagedKVCache
from .quantized_matmul import rope_pair_table
from .rms_norm import rms_norm, rms_norm_fp8


@dataclass(frozen=True)
class DecoderConfig:
    hidden: int
    intermediate: int
    heads: int
    kv_heads: int
    head_dim: int
    layers: int = 1
    group_size: int = 128
    eps: float = 1e-6
    rope_theta: float = 10000.0
    max_positions: int = 4096
    window: Optional[int] = None
    sinks: int = 0


def rope_table(config: DecoderConfig, device="cuda") -> torch.Tensor:
    """(cos, sin) of every position, [max_positions, head_dim / 2, 2] (rope.rs:60-94)."""
    freq = config.rope_theta ** (-torch.arange(0, config.head_dim, 2, dtype=torch.float64)
                                 / config.head_dim)
    ang = torch.arange(config.max_positions, dtype=torch.float64)[:, None] * freq
    ang = ang.repeat_interleave(2, 1)
    return rope_pair_table(ang.cos(), ang.sin()).to(device)


class StepWorkspaces(NamedTuple):
    """What the steps of one graph, or one stream, share: their linears' and their attention's."""
    linear: torch.Tensor
    attend: torch.Tensor


class DecoderLayer:
    """Weights: float tensors in the linears' [out, in] layout, quantized here to 4 bits.

    qkv [(heads + 2 kv_heads) head_dim, hidden] (queries, keys, values; each head's rows in the
    rotary pairs' order (2 i, 2 i + 1), see PagedKVCache.append), out [hidden, heads
    head_dim], gate_up [2 intermediate, hidden] (gate, up), down [hidden, intermediate], and the
    two norms [hidden]."""

    def __init__(self, config: DecoderConfig, qkv: torch.Tensor, out: torch.Tensor,
                 gate_up: torch.Tensor, down: torch.Tensor, norm1: torch.Tensor,
                 norm2: torch.Tensor):
        self.config = config
        quant = lambda w: Int4Linear.from_weight(w, config.group_size)  # noqa: E731
        self.qkv, self.out, self.gate_up, self.down = map(quant, (qkv, out, gate_up, down))
        self.norm1, self.norm2 = norm1, norm2

    @classmethod
    def random(cls, config: DecoderConfig, seed: int = 0, device="cuda",
               dtype: torch.dtype = torch.bfloat16) -> "DecoderLayer":
        g = torch.Generator(device=device).manual_seed(seed)
        make = lambda n, k: torch.randn(n, k, generator=g, device=device) * k ** -0.5  # noqa: E731
        norm = lambda: (1 + 0.1 * torch.randn(config.hidden, generator=g,  # noqa: E731
                                              device=device)).to(dtype)
        c = config
        width = c.heads * c.head_dim
        return cls(c, make(width + 2 * c.kv_heads * c.head_dim, c.hidden), make(c.hidden, width),
                   make(2 * c.intermediate, c.hidden), make(c.hidden, c.intermediate), norm(),
                   norm())

    def step(self, x: torch.Tensor, residual: Optional[torch.Tensor], cache: PagedKVCache,
             block_table: torch.Tensor, seq_ids: torch.Tensor, positions: torch.Tensor,
             seq_lens: torch.Tensor, rope: torch.Tensor,
             workspaces: Optional[StepWorkspaces] = None):
        """x [sequences, hidden]: the layer before's output, residual: the stream it has not been
        added to yet (None: x is the stream).  workspaces: those of `Decoder.new_workspaces` (else
        the stream's).  Returns the same pair for the next layer."""
        c = self.config
        wl, wa = workspaces or (None, None)
        B = x.shape[0]
        if residual is None:
            xq, xs = rms_norm_fp8(x, self.norm1, c.eps)
            residual = x
        else:
            xq, xs, residual = rms_norm_fp8(x, self.norm1, c.eps, residual=residual)
        qkv = self.qkv(xq, xs, out_dtype=x.dtype, workspace=wl).view(B, c.heads + 2 * c.kv_heads, c.head_dim)
        q, k, v = qkv.split((c.heads, c.kv_heads, c.kv_heads), 1)
        q = cache.append(k, v, block_table, seq_ids, positions, q=q, rope=rope)
        o = cache.attend(q, block_table, seq_lens, window=c.window, sinks=c.sinks,
                         workspace=wa)
        x = self.out(o.view(B, c.heads * c.head_dim), workspace=wl)
        xq, xs, residual = rms_norm_fp8(x, self.norm2, c.eps, residual=residual)
        h = swiglu(self.gate_up(xq, xs, out_dtype=x.dtype, workspace=wl))
        return self.down(h, workspace=wl), residual


class Decoder:
    """Layers with a cache each (of the same pages) and a final norm."""

    def __init__(self, config: DecoderConfig, layers: List[DecoderLayer], norm: torch.Tensor,
                 caches: List[PagedKVCache]):
        if not layers or len(layers) != len(caches):
            raise ValueError("at least one layer, and one cache per layer")
        if any(c.page_size != caches[0].page_size or c.pages != caches[0].pages for c in caches):
            raise ValueError("the caches share a block table: as many pages each, of one size")
        self.config, self.layers, self.norm, self.caches = config, layers, norm, caches
        self.rope = rope_table(config, norm.device)

    @classmethod
    def random(cls, config: DecoderConfig, pages: int, page_size: int = 64, seed: int = 0,
               device="cuda", cache_dtype: torch.dtype = torch.bfloat16) -> "Decoder":
        scale = None
        if cache_dtype == torch.float8_e4m3fn:
            scale = torch.full((config.kv_heads,), 0.05, device=device)
        caches = [PagedKVCache.allocate(pages, page_size, config.kv_heads, config.head_dim,
                                        cache_dtype, device, scale, scale)
                  for _ in range(config.layers)]
        layers = [DecoderLayer.random(config, seed + i, device) for i in range(config.layers)]
        norm = torch.ones(config.hidden, dtype=torch.bfloat16, device=device)
        return cls(config, layers, norm, caches)

    def new_workspaces(self, batch: int) -> StepWorkspaces:
        """Workspaces for steps of up to `batch` sequences, one after another."""
        dev = self.norm.device
        need = max(lin.workspace_size(batch) for la in self.layers
                   for lin in (la.qkv, la.out, la.gate_up, la.down))
        return StepWorkspaces(torch.zeros((need + 3) // 4, dtype=torch.int32, device=dev),
                              self.caches[0].new_workspace(self.config.heads))

    def step(self, hidden: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
             workspaces: Optional[StepWorkspaces] = None) -> torch.Tensor:
        """One new token per sequence: hidden [sequences, hidden] its embedding, seq_lens (int32)
        the tokens before it, which its own joins (seq_lens is advanced).  A sequence of
        negative length is padding and stays so.  One that has no room for the token stays as it
        is, too: its length is not advanced, nothing is stored, and its row of the output, which
        attends to nothing, is not a token's.  (No room: max_positions or the block table's
        columns are used up, or the table names no page of the cache at the token's position; with
        the page filled in, the next step goes on.)  Returns the normalised output."""
        B = hidden.shape[0]
        positions, attended = self._advance(seq_lens, block_table)
        seq_ids = torch.arange(B, dtype=torch.int32, device=hidden.device)
        x, residual = hidden, None
        for layer, cache in zip(self.layers, self.caches):
            x, residual = layer.step(x, residual, cache, block_table, seq_ids, positions,
                                     attended, self.rope, workspaces)
        return rms_norm(x, self.norm, self.config.eps, residual=residual)[0]


    def _advance(self, seq_lens: torch.Tensor, block_table: torch.Tensor):
        """Advances seq_lens where the new token has room; (its position or -1, the tokens to
        attend to, its own among them, or 0)."""
        pages, page_size = self.caches[0].pages, self.caches[0].page_size
        end = min(self.config.max_positions, block_table.shape[1] * page_size)
        at = seq_lens.clamp(0, end - 1)
        page = block_table.gather(1, (at // page_size).long()[:, None])[:, 0]
        live = (at == seq_lens) & (page.clamp(0, pages - 1) == page)
        positions = torch.where(live, seq_lens, -1)
        seq_lens += live
        return positions, positions + 1


class DecoderGraph:
    """A decoder's step captured for a batch: replayed with the contents of `hidden`,
    `block_table` and `seq_lens` of the moment; `output` holds the result.

    The graph has workspaces of its own, zeroed once (a captured call without them zeroes one in
    every replay, between kernels that would overlap)."""

    def __init__(self, decoder: Decoder, batch: int, max_pages: int):
        dev = decoder.norm.device
        self.hidden = torch.zeros(batch, decoder.config.hidden, dtype=decoder.norm.dtype,
                                  device=dev)
        self.block_table = torch.full((batch, max_pages), -1, dtype=torch.int32, device=dev)
        self.seq_lens = torch.full((batch,), -1, dtype=torch.int32, device=dev)
        self.workspaces = decoder.new_workspaces(batch)
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):  # padding only: nothing enters the caches
            decoder.step(self.hidden, self.block_table, self.seq_lens, self.workspaces)
        torch.cuda.current_stream(dev).wait_stream(side)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.output = decoder.step(self.hidden, self.block_table, self.seq_lens,
                                       self.workspaces)

    def replay(self) -> torch.Tensor:
        self.graph.replay()
        return self.output


def main() -> None:
    config = DecoderConfig(hidden=4096, intermediate=13824, heads=32, kv_heads=8, head_dim=128,
                           layers=4, max_positions=8192)
    batch, context, page, tokens = 8, 2048, 64, 128
    per = (context + tokens) // page + 1
    decoder = Decoder.random(config, batch * per, page)
    g = DecoderGraph(decoder, batch, per)
    g.block_table.copy_(torch.arange(batch * per, dtype=torch.int32).view(batch, per))
    g.hidden.normal_()
    for warm in (True, False):
        g.seq_lens.fill_(context)
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        for _ in range(tokens):
            g.replay()
        end.record()
        torch.cuda.synchronize()
    ms = start.elapsed_time(end) / tokens
    print(f"{config.layers} layers of {config.hidden}, {batch} sequences from {context} tokens on: "
          f"{ms * 1e3:.0f} us a step, {batch / ms * 1e3:.0f} tokens/s")


__all__ = ["DecoderConfig", "DecoderLayer", "Decoder", "DecoderGraph", "StepWorkspaces",
           "rope_table"]

if __name__ == "__main__":
    main()
