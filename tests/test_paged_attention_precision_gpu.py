"""How near the attention's output is to 64 bits, over all of it.

f16 output has a rounding error of its own, e0.  The weights p, the sums and the exponentials
are to add less than half of it in norm: sqrt(1 + 0.46^2) = 1.1 e0 in all.  (Weights of 11 bits
alone add 2^-11 / sqrt 3 of a weight each, which is 0.8 e0.)"""
import math

import pytest
import torch

from sketchpad_b200 import PagedKVCache
from test_paged_kv_gpu import E4M3, dense, make_cache, make_table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hkv,D,page", [(12, 12, 64, 16), (8, 2, 128, 16), (6, 2, 256, 32),
                                           (8, 2, 80, 12)])
@pytest.mark.parametrize("dtype,cdt", [(torch.float16, torch.float16), (torch.float16, E4M3),
                                       (torch.bfloat16, torch.bfloat16), (torch.bfloat16, E4M3)])
def test_error_is_the_outputs_rounding(hq, hkv, D, page, dtype, cdt):
    lens = [1024, 700, 3000, 33]
    pages = sum(-(-n // page) for n in lens) + 1
    cache = make_cache(pages, page, hkv, D, cdt, seed=D)
    assert isinstance(cache, PagedKVCache)
    table = make_table(lens, page, pages)
    g = torch.Generator("cuda").manual_seed(D + hq)
    q = torch.randn(len(lens), hq, D, generator=g, device="cuda").to(dtype)
    o = cache.attend(q, table, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    ref = torch.empty(o.shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        k, v = dense(cache, table, b, torch.arange(n, device="cuda"))
        p = torch.softmax(q[b].double().reshape(hkv, -1, D) @ k.transpose(1, 2) / math.sqrt(D), -1)
        ref[b] = (p @ v).reshape(hq, D)
    e0 = float((ref.to(dtype).double() - ref).norm())
    assert float((o.double() - ref).norm()) <= 1.1 * e0
