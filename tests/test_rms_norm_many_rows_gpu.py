"""RMS norm at the largest number of rows that it takes: nothing is written before the output."""
import pytest
import torch

from sketchpad_b200 import rms_norm, rms_norm_fp8

pytestmark = pytest.mark.gpu
ROWS = 2 ** 31 - 1
GUARD = 1 << 16  # more rows than the blocks of a launch


@pytest.mark.parametrize("fp8", [False, True])
def test_rows_up_to_31_bits(fp8):
    x = torch.full((ROWS, 1), 0.5, dtype=torch.float16, device="cuda")
    if fp8:
        q, scale = rms_norm_fp8(x, None, 0.0)
        assert bool((q.view(torch.uint8) == 0x7e).all())  # 448
        assert scale.shape == (ROWS,) and float((scale - 1 / 448).abs().max()) < 1e-8
        return
    held = torch.zeros(GUARD + ROWS, dtype=torch.float16, device="cuda")
    y = held[GUARD:].view(ROWS, 1)
    assert rms_norm(x, None, 0.0, out=y) is y
    assert not held[:GUARD].any()
    assert bool((y == 1).all())
