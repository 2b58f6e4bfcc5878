"""The append's numbers of threads per token, which go by the call's length: bit for bit what the
same tokens give in short calls (which have tests against 64 bits)."""
import pytest
import torch

from test_paged_kv_gpu import BF, E4M3, gen, make_cache, make_table, rope_table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [767, 768, 2047, 2048, 2600])
@pytest.mark.parametrize("hq,hkv,D", [(40, 8, 128), (14, 2, 256), (66, 1, 128), (5, 1, 80)])
@pytest.mark.parametrize("cdt", [BF, E4M3])
def test_calls_of_any_length(T, hq, hkv, D, cdt):
    page, pages = 16, T // 16 + 4
    ca, cb = (make_cache(pages, page, hkv, D, cdt) for _ in range(2))
    table = make_table([T + 16], page, pages)
    seq = torch.zeros(T, dtype=torch.int32, device="cuda")
    pos = torch.randperm(T, generator=gen(T), device="cuda").to(torch.int32) + 5
    pos[T // 2] = -1
    qkv = torch.randn(T, hq + 2 * hkv, D, generator=gen(hq), device="cuda").to(BF)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    cs = rope_table(T + 5, D)
    want = torch.cat([ca.append(k[e], v[e], table, seq[e], pos[e], q=q[e], rope=cs)
                      for e in (slice(i, i + 500) for i in range(0, T, 500))])
    got = cb.append(k, v, table, seq, pos, q=q, rope=cs)
    assert torch.equal(got, want) and not got[T // 2].any()
    for x, y in ((ca.k, cb.k), (ca.v, cb.v)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
