"""The token operators in CUDA graphs that outlive the calls around their capture."""
import pytest
import torch

from sketchpad_b200 import Int4Linear, PagedKVCache, _torch
from sketchpad_b200.decoder import Decoder, DecoderConfig, DecoderGraph, DecoderLayer

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def layer(N, K, group=128, seed=0, **kw):
    g = torch.Generator("cuda").manual_seed(seed + N + K)
    q = torch.randint(0, 256, (N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    s = (torch.rand(K // group, N, generator=g, device="cuda") / 64).half()
    return Int4Linear(q, s, group_size=group, **kw)


def occupy(nbytes):
    """Tensors of the sizes of freed workspaces, none of their bytes zero."""
    return [torch.full((n,), 0x5a, dtype=torch.uint8, device="cuda")
            for n in (nbytes, nbytes, nbytes // 2, nbytes // 2) for _ in range(8)]


def test_linear_captured_on_a_stream_that_is_used_again():
    small, large = layer(1024, 16384, 64), layer(40000, 16384, 64)
    assert large.workspace_size(32) > small.workspace_size(16)
    x = torch.randn(13, 16384, device="cuda").to(BF)
    want = [small(x * f) for f in (1, 2, 3)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    xin, out = torch.zeros_like(x), torch.zeros_like(want[0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        small(xin, out=out)
        s.synchronize()
        with torch.cuda.graph(g, stream=s):
            small(xin, out=out)
        held = [large(torch.randn(32, 16384, device="cuda").to(BF))]
        s.synchronize()
        held += occupy(small.workspace_size(16))
        for f, w in zip((1, 2, 3), want):
            xin.copy_(x * f)
            out.zero_()
            g.replay()
            small(x)  # the stream's own calls between replays
            s.synchronize()
            assert torch.equal(out, w)
    assert all(bool((t == 0x5a).all()) for t in held[1:])


def test_attention_captured_on_a_stream_that_is_used_again():
    gen = torch.Generator("cuda").manual_seed(3)
    k, v = (torch.randn(130, 16, 2, 128, generator=gen, device="cuda").to(BF) for _ in range(2))
    cache = PagedKVCache(k, v)
    table = torch.randperm(130, generator=gen, device="cuda").to(torch.int32)[None, :128].contiguous()
    lens = torch.tensor([2000], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 4, 128, generator=gen, device="cuda").to(BF)
    qw = torch.randn(1, 32, 128, generator=gen, device="cuda").to(BF)
    assert cache.workspace_size(32) > cache.workspace_size(4)
    want = [cache.attend(q, table, lens - d) for d in (0, 1, 700)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    ln, out = lens.clone(), torch.zeros_like(q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        cache.attend(q, table, ln, out=out)
        s.synchronize()
        with torch.cuda.graph(g, stream=s):
            cache.attend(q, table, ln, out=out)
        cache.attend(qw, table, lens)
        s.synchronize()
        held = occupy(cache.workspace_size(4))
        for d, w in zip((0, 1, 700), want):
            ln.copy_(lens - d)
            out.zero_()
            g.replay()
            cache.attend(q, table, lens)
            s.synchronize()
            assert torch.equal(out, w)
    assert all(bool((t == 0x5a).all()) for t in held)


def test_bias_of_a_first_call_under_capture():
    # the cast to the output's type is not the graph's: calls before the first replay have it too
    bias = torch.randn(512, device="cuda")
    lin = layer(512, 1024, bias=bias)
    plain = layer(512, 1024)
    x = torch.randn(3, 1024, device="cuda").to(BF)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = lin(x)
        junk = [torch.zeros(512, dtype=BF, device="cuda") for _ in range(8)]
    err = (lin(x).double() - plain(x, out_dtype=torch.float32).double() - bias.to(BF).double()).abs()
    bound = 2.0 ** -7 * (plain(x, out_dtype=torch.float32).double().abs() + bias.double().abs())
    assert bool((err <= bound).all())
    g.replay()
    assert torch.equal(out, lin(x)) and len(junk) == 8


def test_bias_is_the_layers_own():
    # like the weights: later changes of the given tensor reach no output type
    bias = torch.randn(512, device="cuda")
    lin = layer(512, 1024, bias=bias)
    x = torch.randn(3, 1024, device="cuda").to(BF)
    types = (torch.float32, torch.float16, BF)
    before = [lin(x, out_dtype=t) for t in types]
    other = layer(512, 1024, bias=bias.clone())
    bias.add_(1000)
    assert all(torch.equal(lin(x, out_dtype=t), b) for t, b in zip(types, before))
    assert all(torch.equal(other(x, out_dtype=t), b) for t, b in zip(types, before))
    assert torch.equal(lin.bias, bias - 1000) or float((lin.bias - (bias - 1000)).abs().max()) < 1e-3


def test_a_captured_step_zeroes_no_workspaces(monkeypatch):
    c = DecoderConfig(hidden=512, intermediate=768, heads=8, kv_heads=2, head_dim=64, layers=2,
                      group_size=64, max_positions=64)
    dec = Decoder.random(c, pages=8, page_size=16)
    made, get = [], _torch.Workspaces.get

    def record(self, *a):
        made.append(a)
        return get(self, *a)

    monkeypatch.setattr(_torch.Workspaces, "get", record)
    g = DecoderGraph(dec, 2, 4)
    assert not made
    monkeypatch.undo()
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    g.block_table.copy_(table)
    g.seq_lens.zero_()
    hidden = torch.randn(20, 2, c.hidden, device="cuda").to(BF)
    outs = []
    for h in hidden:
        g.hidden.copy_(h)
        outs.append(g.replay().clone())
    w = g.workspaces
    torch.cuda.synchronize()
    assert not w.linear[:1 << 16].any() and not w.attend[:1 << 18].any()  # the counters
    for h, out in zip(hidden, outs):
        assert torch.equal(dec.step(h, table, lens), out)


def test_a_graph_of_an_f16_decoder():
    c = DecoderConfig(hidden=256, intermediate=256, heads=4, kv_heads=2, head_dim=64,
                      group_size=64, max_positions=64)
    HF = torch.float16
    k, v = (torch.zeros(4, 16, 2, 64, dtype=HF, device="cuda") for _ in range(2))
    dec = Decoder(c, [DecoderLayer.random(c, dtype=HF)], torch.ones(256, dtype=HF, device="cuda"),
                  [PagedKVCache(k, v)])
    g = DecoderGraph(dec, 1, 4)
    assert g.hidden.dtype == g.output.dtype == HF
    g.block_table.copy_(torch.arange(4, dtype=torch.int32)[None])
    g.seq_lens.zero_()
    lens = torch.zeros(1, dtype=torch.int32, device="cuda")
    for h in torch.randn(5, 1, 256, device="cuda").to(HF):
        g.hidden.copy_(h)
        out = g.replay().clone()
        assert torch.equal(dec.step(h, g.block_table, lens), out)
