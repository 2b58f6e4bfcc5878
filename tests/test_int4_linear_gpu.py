"""4-bit linear against y = x . (s (q - z))^T in 64 bits.

Bound per output, with A = sum |s (q - z) x| over its inputs: the products are exact in the MMA;
its accumulator takes at most 128 / 16 steps per group, each within 2^-22 of the partial sum;
the groups' sums and the joins over warps and blocks are f32 adds and multiplies, K / group + 64
of them at most in a row.  So |err| <= A (8 * 2^-22 + (K / group + 64) 2^-24), then the output's
own rounding (2^-8 bf16, 2^-11 f16, none f32)."""
import numpy as np
import pytest
import torch

from sketchpad_b200 import Int4Linear, SketchpadError, rms_norm_fp8

pytestmark = pytest.mark.gpu
ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
E4M3 = torch.float8_e4m3fn


def weight(N, K, group, zeros, sdt, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 3 * N + K)
    q = torch.randint(0, 256, (N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    s = ((0.5 + torch.rand(K // group, N, generator=g, device="cuda")) / 64).to(sdt)
    z = torch.randint(0, 16, (K // group, N), generator=g, device="cuda",
                      dtype=torch.uint8) if zeros else None
    return q, s, z


def values(q, s, z, group):
    v = torch.stack((q & 15, q >> 4), -1).reshape(q.shape[0], -1).double()
    zz = 8.0 if z is None else z.t().double().repeat_interleave(group, 1)
    return (v - zz) * s.t().double().repeat_interleave(group, 1)


def check(y, x, w, group, bias=None):
    ref, a = x.double() @ w.t(), x.double().abs() @ w.t().abs()
    if bias is not None:
        ref, a = ref + bias.double(), a + bias.double().abs()
    K = w.shape[1]
    bound = a * (8 * 2.0 ** -22 + (K / group + 64) * 2.0 ** -24) + ref.abs() * ROUND[y.dtype]
    err = (y.double() - ref).abs()
    if y.dtype == torch.float16:
        bound = bound + 2.0 ** -25
    assert y.shape == ref.shape and bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("M", [1, 2, 7, 8, 9, 16, 17, 32, 33, 70])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True), (256, False)])
def test_rows(M, dtype, group, zeros):
    N, K = 200, 1024
    q, s, z = weight(N, K, group, zeros, dtype)
    x = torch.randn(M, K, device="cuda", generator=torch.Generator("cuda").manual_seed(M)).to(dtype)
    lin = Int4Linear(q, s, z, group_size=group)
    check(lin(x), x, values(q, s, z, group), group)


@pytest.mark.parametrize("N,K,group", [(1, 32, 32), (16, 32, 32), (5, 96, 32), (33, 224, 32),
                                       (1001, 2016, 32), (257, 64, 64), (48, 192, 64),
                                       (100, 4096, 4096), (16, 13824, 128), (4096, 4096, 128),
                                       (2048, 28672, 64), (8, 131072, 128)])
@pytest.mark.parametrize("zeros", [False, True])
def test_shapes(N, K, group, zeros):
    q, s, z = weight(N, K, group, zeros, torch.float16)
    g = torch.Generator("cuda").manual_seed(N)
    for M in (1, 12, 32):
        x = torch.randn(M, K, device="cuda", generator=g).to(torch.bfloat16)
        lin = Int4Linear(q, s, z, group_size=group)
        check(lin(x, out_dtype=torch.float32), x, values(q, s, z, group), group)


@pytest.mark.parametrize("M", [1, 5, 20])
@pytest.mark.parametrize("odt", [torch.bfloat16, torch.float16, torch.float32])
def test_e4m3_rows_and_bias(M, odt):
    N, K, group = 300, 640, 64
    q, s, z = weight(N, K, group, True, torch.bfloat16)
    g = torch.Generator("cuda").manual_seed(M)
    h = torch.randn(M, K, device="cuda", generator=g).to(torch.bfloat16)
    xq, xs = rms_norm_fp8(h, None)
    bias = torch.randn(N, device="cuda", generator=g)
    lin = Int4Linear(q, s, z, group_size=group, bias=bias)
    y = lin(xq, xs, out_dtype=odt)
    check(y, xq.double() * xs.double()[:, None], values(q, s, z, group), group, bias.to(odt))
    assert lin(xq, xs).dtype == torch.bfloat16


def test_dequantize_is_exact():
    for N, K, group in ((37, 96, 32), (50, 192, 64), (20, 512, 256)):
        for zeros in (False, True):
            for sdt in (torch.float16, torch.bfloat16):
                q, s, z = weight(N, K, group, zeros, sdt)
                w = Int4Linear(q, s, z, group_size=group).dequantize()
                assert torch.equal(w.double(), values(q, s, z, group))


def test_from_weight_and_from_gguf():
    g = torch.Generator("cuda").manual_seed(5)
    w = torch.randn(70, 256, generator=g, device="cuda")
    for symmetric in (True, False):
        lin = Int4Linear.from_weight(w, 64, symmetric)
        wd = lin.dequantize()
        r = w.reshape(70, 4, 64)
        step = (r.abs().amax(-1) / 7 if symmetric else
                (r.amax(-1).clamp(min=0) - r.amin(-1).clamp(max=0)) / 15)
        # half a step from rounding, another half where the zero point's rounding cuts an end,
        # and the f16 scale's own rounding over 15 steps
        slack = step[..., None] * ((0.5 if symmetric else 1.0) + 16 * 2.0 ** -11)
        assert bool(((wd - w).reshape(70, 4, 64).abs() <= slack).all())
    rng = np.random.default_rng(0)
    blocks = rng.integers(0, 256, (24, 3, 18), dtype=np.uint8)
    d = rng.uniform(-0.02, 0.02, (24, 3)).astype(np.float16)
    d[0, 0], d[0, 1] = 6e-8, 0.0
    blocks[..., :2] = d.view(np.uint8).reshape(24, 3, 2)
    lin = Int4Linear.from_gguf_q4_0(blocks.tobytes(), 24, 96)
    nib = np.concatenate((blocks[..., 2:] & 15, blocks[..., 2:] >> 4), -1).astype(np.float32)
    ref = (d.astype(np.float32)[..., None] * (nib - 8)).reshape(24, 96)
    assert np.array_equal(lin.dequantize().cpu().numpy(), ref)


def test_strided_and_unaligned_rows():
    N, K, group = 64, 256, 128
    q, s, z = weight(N, K, group, False, torch.bfloat16)
    lin, w = Int4Linear(q, s, z, group_size=group), values(q, s, z, group)
    big = torch.randn(6, 5, 3 * K, device="cuda").to(torch.bfloat16)
    for x in (big[:, 0, :K], big[:, 1, 8:8 + K], big[:, 2, 3:3 + K], big[0, :, K:2 * K],
              big[:, :, :K], big[0, 0, ::3], big[0, 0, :K].expand(4, K)):
        y = lin(x)
        assert y.shape == (*x.shape[:-1], N)
        check(y.reshape(-1, N), x.reshape(-1, K), w, group)


def test_values_that_stand_out():
    # a NaN or an infinity in one row of x stays in that row; values near the types' ends
    q, s, z = weight(40, 256, 64, True, torch.float16)
    w = values(q, s, z, 64)
    x = torch.randn(4, 256, device="cuda").to(torch.bfloat16)
    x[1, 5], x[2, 100] = float("nan"), float("inf")
    x[3] *= 1e30
    y = Int4Linear(q, s, z, group_size=64)(x, out_dtype=torch.float32)
    assert torch.isnan(y[1]).all()
    assert not torch.isfinite(y[2][w[:, 100] != 0]).any()
    check(y[[0, 3]], x[[0, 3]], w, 64)


def test_repeats_bit_for_bit_and_streams():
    q, s, z = weight(4096, 4096, 128, False, torch.bfloat16)
    lin = Int4Linear(q, s, z, group_size=128)
    x = torch.randn(3, 4096, device="cuda").to(torch.bfloat16)
    a = lin(x)
    assert all(torch.equal(a, lin(x)) for _ in range(5))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        x2 = x * 2
        b = lin(x2)
    side.synchronize()
    assert torch.equal(b, a * 2)
    assert lin(x[:0]).shape == (0, 4096)


def test_refusals():
    q, s, z = weight(32, 256, 64, True, torch.float16)
    for args, kw in (((q, s, z), dict(group_size=32)), ((q, s.float(), z), dict(group_size=64)),
                     ((q, s, z.int()), dict(group_size=64)), ((q.int(), s, z), dict(group_size=64)),
                     ((q, s, z), dict(group_size=64, bias=s[0, :5]))):
        with pytest.raises(ValueError):
            Int4Linear(*args, **kw)
    for group in (0, 48, 96, 512):
        with pytest.raises(SketchpadError):
            Int4Linear(q, s, z, group_size=group)
    lin = Int4Linear(q, s, z, group_size=64)
    x = torch.randn(2, 256, device="cuda")
    h, scale = x.half(), torch.ones(2, device="cuda")
    with pytest.raises(TypeError):
        lin(x)
    for bad in (lambda: lin(h[:, :128]), lambda: lin(h, scale), lambda: lin(x.to(E4M3)),
                lambda: lin(x.to(E4M3), scale[:1]), lambda: lin(x.to(E4M3), scale.half()),
                lambda: lin(h, out=torch.empty(2, 31, device="cuda", dtype=torch.float16)),
                lambda: lin(h.cpu())):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("M", [40, 65, 96])
@pytest.mark.parametrize("N,K,group", [(144, 8192, 32), (1000, 13824, 128)])
def test_more_rows_than_a_launch_takes(M, N, K, group):
    """Launches that follow one another in a call share its workspace: bit for bit what calls of
    their rows give."""
    q, s, z = weight(N, K, group, True, torch.float16)
    layer = Int4Linear(q, s, z, group_size=group)
    x = torch.randn(M, K, generator=torch.Generator("cuda").manual_seed(M), device="cuda").half()
    want = torch.cat([layer(x[i:i + 32]) for i in range(0, M, 32)])
    for _ in range(3):
        assert torch.equal(layer(x), want)
