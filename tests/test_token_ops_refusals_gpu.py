"""Calls of the token operators that are refused on the host, before anything is launched."""
import pytest
import torch

from sketchpad_b200 import Int4Linear, PagedKVCache, rms_norm

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def test_workspaces_that_are_not_contiguous():
    lin = Int4Linear(torch.zeros(64, 64, dtype=torch.uint8, device="cuda"),
                     torch.ones(1, 64, dtype=torch.float16, device="cuda"), group_size=128)
    w = torch.zeros(lin.workspace_size(1) // 4, 2, dtype=torch.int32, device="cuda")[:, 0]
    x = torch.zeros(1, 128, dtype=BF, device="cuda")
    with pytest.raises(ValueError):
        lin(x, workspace=w)
    assert not lin(x, workspace=w.contiguous()).any()
    t = torch.zeros(2, 16, 1, 64, dtype=BF, device="cuda")
    cache = PagedKVCache(t, t.clone())
    w = torch.zeros(cache.workspace_size(1) // 4 + 1, 2, dtype=torch.int32, device="cuda")[:, 0]
    q = torch.zeros(1, 1, 64, dtype=BF, device="cuda")
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    n = torch.ones(1, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        cache.attend(q, table, n, workspace=w)
    assert not cache.attend(q, table, n, workspace=w.contiguous()).any()


def test_scales_that_the_entry_would_replace():
    t = torch.randn(2, 16, 1, 64, device="cuda").to(BF)
    cache = PagedKVCache(t, t.clone())
    q = torch.randn(1, 1, 64, device="cuda").to(BF)
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    n = torch.full((1,), 9, dtype=torch.int32, device="cuda")
    for scale in (0.0, -0.125, float("nan"), float("inf"), 1e-45):
        with pytest.raises(ValueError):
            cache.attend(q, table, n, scale=scale)
    assert torch.equal(cache.attend(q, table, n), cache.attend(q, table, n, scale=0.125))


def test_norm_and_stream_into_one_memory():
    x, r = torch.randn(2, 3, 64, device="cuda").to(BF)
    buf = torch.empty_like(x)
    for kw in (dict(out=buf, residual_out=buf), dict(out=x, residual_out=x)):
        with pytest.raises(ValueError):
            rms_norm(x, None, residual=r, **kw)
    y, s = rms_norm(x, None, residual=r, out=buf)
    assert y is buf and torch.equal(s, x + r)
