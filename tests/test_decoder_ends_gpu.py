"""A decoder's sequences that cannot take another token: at the rotary table's end, at the block
table's, and where no page is there."""
import pytest
import torch

from sketchpad_b200.decoder import Decoder, DecoderConfig, DecoderGraph

pytestmark = pytest.mark.gpu


def make(max_positions, pages=12, layers=2, page_size=8):
    c = DecoderConfig(hidden=256, intermediate=256, heads=4, kv_heads=2, head_dim=64, layers=layers,
                      group_size=64, max_positions=max_positions)
    return Decoder.random(c, pages=pages, page_size=page_size)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("max_positions,cols,end", [(20, 3, 20), (64, 2, 16), (16, 2, 16)])
@pytest.mark.parametrize("graph", [False, True])
def test_a_full_sequence_stays_where_it_is(max_positions, cols, end, graph):
    dec, alone = make(max_positions), make(max_positions)
    table = torch.arange(2 * cols, dtype=torch.int32, device="cuda").view(2, cols)
    for cache in dec.caches:  # what an earlier owner of the pages left
        cache.k.fill_(float("nan"))
        cache.v.fill_(float("nan"))
    g = None
    if graph:
        g = DecoderGraph(dec, 2, cols)
        g.block_table.copy_(table)
    lens = g.seq_lens if graph else ints(0, 0)
    lens.copy_(ints(0, 6 - end))  # the second is padding at first ...
    one = ints(0)
    gen = torch.Generator("cuda").manual_seed(0)
    for step in range(end + 4):
        if step == 6:
            lens[1] = 0           # ... and joins at the seventh step
        hidden = torch.randn(2, 256, generator=gen, device="cuda").to(torch.bfloat16)
        if graph:
            g.hidden.copy_(hidden)
            out = g.replay()
        else:
            out = dec.step(hidden, table, lens)
        want = [min(step + 1, end), min(step - 5, end) if step >= 6 else 6 - end]
        assert lens.tolist() == want
        assert torch.isfinite(out).all()
        if step >= 6:  # the second is not moved by the first one's end
            assert torch.equal(out[1:], alone.step(hidden[1:], table[1:], one))
    for cache in dec.caches:  # nothing was stored behind the end
        k = cache.k[table[0].long()].reshape(-1, 2, 64)
        assert torch.isfinite(k[:end]).all() and torch.isnan(k[end:]).all()


def test_a_sequence_waits_for_its_page():
    dec, alone = make(64), make(64)
    table, full = ints(3, -1).view(1, 2), ints(3, 5).view(1, 2)
    lens, lens1 = ints(0), ints(0)
    gen = torch.Generator("cuda").manual_seed(0)
    for step in range(14):
        hidden = torch.randn(1, 256, generator=gen, device="cuda").to(torch.bfloat16)
        if step in (9, 10):       # no page for the ninth token yet, then one outside the pool
            before = [c.k.clone() for c in dec.caches]
            out = dec.step(hidden, ints(3, 12).view(1, 2) if step == 10 else table, lens)
            assert lens.tolist() == [8] and torch.isfinite(out).all()
            assert all(torch.equal(a, c.k) for a, c in zip(before, dec.caches))
            continue
        if step == 8:
            continue
        out = dec.step(hidden, full if step > 10 else table, lens)
        assert torch.equal(out, alone.step(hidden, full, lens1))
    assert lens.tolist() == [11]
