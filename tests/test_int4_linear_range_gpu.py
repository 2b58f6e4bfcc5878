"""The 4-bit linear at the ends of the types' ranges, and with channels far above the rest.

x is staged in f16, a row's largest value at 2^14 or above: what f16 cannot hold is at most
2^-25 / 2^14 = 2^-39 of the row's largest value per input; 2^-35 max|x| sum |w| in all is allowed.
The rest is the bound of the ordinary sizes, and where the results come near f32's subnormals
their quantum, once per slab of the inputs (64 at most here)."""
import pytest
import torch

from sketchpad_b200 import Int4Linear
from test_int4_linear_gpu import values, weight

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def check(y, x, w, group, quantum=0.0):
    assert y.dtype == F32
    xd = x.double()
    ref, a = xd @ w.t(), xd.abs() @ w.t().abs()
    staged = 2.0 ** -35 * xd.abs().amax(1)[:, None] * w.abs().sum(1)
    bound = a * (8 * 2.0 ** -22 + (w.shape[1] / group + 64) * 2.0 ** -24) + staged + \
        ref.abs() * 2.0 ** -24 + quantum
    err = (y.double() - ref).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("N,K,group,zeros", [(40, 256, 64, True), (64, 16384, 32, False),
                                             (5120, 13824, 128, True)])
@pytest.mark.parametrize("exponent", [-132, -126, -100, 104, 117, 118, 119, 122])
def test_rows_at_the_ends_of_bf16(N, K, group, zeros, exponent):
    q, s, z = weight(N, K, group, zeros, HF)
    if exponent > 100:
        s = s / 64  # sums stay within f32
    x = torch.rand(11, K, device="cuda", generator=torch.Generator("cuda").manual_seed(1)) - 0.5
    x[:, 0] = 1  # the row's largest
    x = (x.double() * 2.0 ** exponent).to(BF)
    x[1] = 0
    x[1, 3] = 2.0 ** exponent
    w = values(q, s, z, group)
    if exponent > 100:
        w = values(q, s, z, group)
        assert float((x.double().abs() @ w.t().abs()).max()) < 2.0 ** 127
    y = Int4Linear(q, s, z, group_size=group)(x, out_dtype=F32)
    assert torch.isfinite(y).all()
    check(y, x, w, group, 65 * 2.0 ** -150 if exponent <= -126 else 0.0)


def test_last_exponents_of_bf16():
    # single inputs, so that the products stay within f32
    q, s, z = weight(40, 256, 64, True, BF)
    s = (s.float() * 2.0 ** -20).to(BF)
    w = values(q, s, z, 64)
    x = torch.zeros(10, 256, device="cuda", dtype=BF)
    for r in range(10):
        x[r, 7 * r] = 1.5 * 2.0 ** (118 + r)
    check(Int4Linear(q, s, z, group_size=64)(x, out_dtype=F32), x, w, 64)


@pytest.mark.parametrize("M", [1, 6, 20])
@pytest.mark.parametrize("group,zeros", [(32, False), (64, True), (128, True), (128, False)])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("power", [10, 13, 16, 20])
def test_channels_far_above_the_rest(M, group, zeros, dtype, power):
    # the large channels meet weights that equal the zero point in every other output: there
    # they count nothing, however large
    N, K = 130, 1024
    q, s, z = weight(N, K, group, zeros, HF)
    big = [5, 130, 517, 1022]
    zp = torch.full((K // group, N), 8, dtype=torch.uint8, device="cuda") if z is None else z
    for k in big:
        n = torch.arange(0, N, 2, device="cuda")
        v = zp[k // group, n]
        old = q[n, k // 2]
        q[n, k // 2] = ((old & 0xf0) | v) if k % 2 == 0 else ((old & 0x0f) | (v << 4))
    x = torch.randn(M, K, device="cuda", generator=torch.Generator("cuda").manual_seed(power))
    scale = 1.0 if dtype == BF else 2.0 ** -min(power - 10, 8)
    x = x * scale
    x[:, big] = scale * 2.0 ** power * torch.tensor([1.0, -0.75, 1.25, 0.5], device="cuda")
    x = x.to(dtype)
    assert torch.isfinite(x.float()).all()
    w = values(q, s, z, group)
    assert not w[::2][:, big].any()
    check(Int4Linear(q, s, z, group_size=group)(x, out_dtype=F32), x, w, group)
