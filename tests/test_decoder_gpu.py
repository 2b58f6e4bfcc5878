"""The token operators together: decoder steps against the layers' formulas in 64 bits.

The reference forms the same e4m3 rows.  A bf16 rounding before one (2^-9) moves about 2^-9 /
2^-4 = 3 % of the values over to the next e4m3 value, 2^-4 to 2^-3 away: sqrt(0.03) * 2^-4 = 1.1 %
of the row's 2-norm per norm, two norms a layer, three layers and the bf16 roundings between
them: sqrt(6) * 1.1 % + 6 * 0.2 % < 4 %, held to 6 %.  (An e4m3 cache moves keys and values over in the
same way, which this does not count: there the reference attends to the rows that the cache
holds, whose own rounding the cache's tests check.)"""
import math

import pytest
import torch

from sketchpad_b200.decoder import Decoder, DecoderConfig, DecoderGraph

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def norm(x, w, eps):
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()


def to_e4m3(y):
    s = y.abs().amax(-1, keepdim=True) / 448
    s = torch.where(s == 0, 1.0, s)
    return (y / s).clamp(-448, 448).float().to(E4M3).double() * s


def plain_step(dec, hidden, lens, kv, stored):
    """hidden [B, H] f64; kv[layer][b] = lists of (k, v) rows; lens before the step."""
    c = dec.config
    x, res = torch.zeros_like(hidden), hidden
    for i, layer in enumerate(dec.layers):
        res = res + x
        h = to_e4m3(norm(res, layer.norm1, c.eps)) @ layer.qkv.dequantize().double().t()
        h = h.view(-1, c.heads + 2 * c.kv_heads, c.head_dim)
        out = torch.zeros(len(lens), c.heads * c.head_dim, dtype=torch.float64, device="cuda")
        for b, n in enumerate(lens):
            if n < 0:
                continue
            z = torch.view_as_complex(dec.rope[n].double())
            turn = lambda t: torch.view_as_real(torch.view_as_complex(  # noqa: E731
                t.reshape(t.shape[0], -1, 2).contiguous()) * z).reshape(t.shape)
            q, k, v = h[b].split((c.heads, c.kv_heads, c.kv_heads))
            kv[i][b].append(stored(i, b, n) if stored else (turn(k), v))
            ks = torch.stack([t[0] for t in kv[i][b]], 1)  # [hkv, n, D]
            vs = torch.stack([t[1] for t in kv[i][b]], 1)
            m = n + 1
            keep = torch.arange(m, device="cuda")
            if c.window:
                keep = keep[(keep >= m - c.window) | (keep < c.sinks)]
            ks, vs = ks[:, keep], vs[:, keep]
            qq = turn(q).reshape(c.kv_heads, -1, c.head_dim)
            p = torch.softmax(qq @ ks.transpose(1, 2) / math.sqrt(c.head_dim), -1)
            out[b] = (p @ vs).reshape(-1)
        res = res + out @ layer.out.dequantize().double().t()
        h = to_e4m3(norm(res, layer.norm2, c.eps)) @ layer.gate_up.dequantize().double().t()
        gate, up = h.chunk(2, -1)
        x = (torch.nn.functional.silu(gate) * up) @ layer.down.dequantize().double().t()
    return norm(res + x, dec.norm, c.eps)


@pytest.mark.parametrize("cache_dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("window,sinks", [(None, 0), (5, 2)])
def test_steps(cache_dtype, window, sinks):
    c = DecoderConfig(hidden=256, intermediate=384, heads=8, kv_heads=2, head_dim=64, layers=3,
                      group_size=64, max_positions=64, window=window, sinks=sinks)
    dec = Decoder.random(c, pages=12, page_size=8, cache_dtype=cache_dtype)
    B = 4
    table = torch.randperm(12, generator=torch.Generator().manual_seed(0))[:12].view(B, 3)
    table = table.to(torch.int32).cuda()
    start = [0, 0, -1, 0]  # the third sequence is padding
    lens = torch.tensor(start, dtype=torch.int32, device="cuda")
    kv = [[[] for _ in range(B)] for _ in range(c.layers)]

    def stored(i, b, n):
        cache, at = dec.caches[i], (int(table[b, n // 8]), n % 8)
        return tuple(t[at].float().double() * 0.05 for t in (cache.k, cache.v))

    g = torch.Generator("cuda").manual_seed(1)
    for step in range(18):
        hidden = torch.randn(B, c.hidden, generator=g, device="cuda").to(torch.bfloat16)
        before = lens.tolist()
        out = dec.step(hidden, table, lens)
        ref = plain_step(dec, hidden.double(), before, kv,
                         stored if cache_dtype == E4M3 else None)
        assert lens.tolist() == [n + 1 if n >= 0 else n for n in before]
        for b in (0, 1, 3):
            err = (out[b].double() - ref[b]).norm() / ref[b].norm()
            assert float(err) < 0.06, (step, b, float(err))


def test_graph_replays_what_the_steps_compute():
    c = DecoderConfig(hidden=256, intermediate=256, heads=4, kv_heads=2, head_dim=64, layers=2,
                      group_size=32, max_positions=256)
    dec = Decoder.random(c, pages=24, page_size=16)
    g = DecoderGraph(dec, 3, 4)
    g.block_table.copy_(torch.arange(12, dtype=torch.int32).view(3, 4))
    g.seq_lens.copy_(torch.tensor([0, 0, -1], dtype=torch.int32))
    table = torch.arange(12, 24, dtype=torch.int32, device="cuda").view(3, 4)
    lens = torch.tensor([0, 0, -1], dtype=torch.int32, device="cuda")
    for step in range(40):
        hidden = torch.randn(3, c.hidden, device="cuda").to(torch.bfloat16)
        g.hidden.copy_(hidden)
        a = g.replay()[:2].clone()
        b = dec.step(hidden, table, lens)[:2]
        assert torch.equal(a, b) and torch.equal(g.seq_lens, lens)
