"""RMS norm (with residual, in the stream's type or e4m3) against its formula in 64 bits.

Bounds, element by element.  f32 arithmetic: the sum of squares of a row is at most 16 terms per
thread and 10 shuffle levels, halved by the square root, then five more roundings: below 32
half-ulps, 32 * 2^-24 < 2e-6 relative.  Then one rounding to the output: 2^-8 (bf16), 2^-11
(f16; 2^-25 absolute where subnormal), 2^-4 (e4m3; 2^-10 where subnormal)."""
import pytest
import torch

from sketchpad_b200 import rms_norm, rms_norm_fp8

pytestmark = pytest.mark.gpu
F32 = 2e-6
HALF = {torch.float32: (0.0, 0.0), torch.bfloat16: (2.0 ** -8, 0.0),
        torch.float16: (2.0 ** -11, 2.0 ** -25)}
E4M3 = torch.float8_e4m3fn


def inputs(rows, n, dtype, residual, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + rows * 7 + n)
    x = torch.randn(rows, n, generator=g, device="cuda").to(dtype)
    w = (1 + 0.2 * torch.randn(n, generator=g, device="cuda")).to(dtype)
    r = (3 * torch.randn(rows, n, generator=g, device="cuda")).to(dtype) if residual else None
    return x, w, r


def formula(x, w, r, eps):
    s = x if r is None else (x.double() + r.double()).to(x.dtype)
    d = s.double()
    y = d / (d.square().mean(-1, keepdim=True) + eps).sqrt()
    return (y if w is None else y * w.double()), s


def check(y, ref, dtype, extra=0.0):
    rel, absolute = HALF[dtype]
    err = (y.double() - ref).abs()
    bound = (rel + F32 + extra) * ref.abs() + absolute
    assert bool((err <= bound).all()), float((err - bound).max())


def check_fp8(q, scale, ref):
    amax = ref.abs().amax(-1)
    s = torch.where(amax == 0, 1.0, amax / 448)
    assert bool(((scale.double() - s).abs() <= 2 * F32 * s).all())
    v = ref / s[..., None]
    err = (q.double() - v).abs()
    bound = torch.maximum(v.abs() * 2.0 ** -4, torch.full_like(v, 2.0 ** -10)) + 448 * 4 * F32
    assert bool((err <= bound).all()), float((err - bound).max())


SIZES = [(1, 1), (1, 4096), (3, 7), (5, 8), (2, 640), (17, 1031), (64, 5120), (9, 2051),
         (4, 8200), (2, 16384), (2, 8193), (3, 32768), (1, 40000)]


@pytest.mark.parametrize("rows,n", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm(rows, n, dtype, residual):
    x, w, r = inputs(rows, n, dtype, residual)
    ref, s = formula(x, w, r, 1e-6)
    got = rms_norm(x, w, 1e-6, residual=r)
    y = got[0] if residual else got
    # rows beyond 16 elements per thread add n / 1024 terms to a thread's sum
    check(y, ref, dtype, extra=max(0, n // 1024 - 16) * 2.0 ** -25)
    if residual:
        assert torch.equal(got[1], s)


@pytest.mark.parametrize("rows,n", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm_fp8(rows, n, dtype, residual):
    x, w, r = inputs(rows, n, dtype, residual, 1)
    ref, s = formula(x, w, r, 1e-5)
    got = rms_norm_fp8(x, w, 1e-5, residual=r)
    assert got[0].dtype == E4M3 and got[1].shape == (rows,)
    check_fp8(got[0], got[1], ref)
    if residual:
        assert torch.equal(got[2], s)


def test_in_place_and_without_weight():
    x, w, r = inputs(33, 512, torch.bfloat16, True)
    ref, s = formula(x, None, r, 1e-6)
    stream = r.clone()
    xin = x.clone()
    y, out = rms_norm(xin, None, 1e-6, residual=stream, out=xin, residual_out=stream)
    assert y is xin and out is stream and torch.equal(stream, s)
    check(y, ref, torch.bfloat16)
    for n in (8193, 40000):  # the rows of the other two paths, in place
        x, w, r = inputs(2, n, torch.float32, True)
        ref, s = formula(x, w, r, 1e-6)
        y, out = rms_norm(x, w, 1e-6, residual=r, out=x, residual_out=r)
        assert torch.equal(r, s)
        check(y, ref, torch.float32, extra=n // 1024 * 2.0 ** -25)


def test_strided_rows_and_leading_dimensions():
    big = torch.randn(2, 3, 1000, device="cuda").to(torch.bfloat16)
    w = torch.ones(300, device="cuda", dtype=torch.bfloat16)
    for lo in (0, 8, 1, 333):  # aligned and unaligned column slices
        x = big[:, :, lo:lo + 300]
        y = rms_norm(x, w)
        assert y.shape == (2, 3, 300) and y.is_contiguous()
        check(y, formula(x, w, None, 1e-6)[0], torch.bfloat16)
        q, s = rms_norm_fp8(x, w)
        assert s.shape == (2, 3)
        check_fp8(q, s, formula(x, w, None, 1e-6)[0])


def test_zero_nan_and_infinite_rows():
    x = torch.randn(5, 4096, device="cuda")
    x[0] = 0
    x[1, 7] = float("nan")
    x[2, 9] = float("inf")
    x[3] = 1e-30
    q, s = rms_norm_fp8(x, None)
    y = rms_norm(x, None)
    assert s[0] == 1 and not q[0].float().any() and not y[0].any()
    assert torch.isnan(s[1]) and torch.isnan(q[1].float()).all() and torch.isnan(y[1]).all()
    # 1 / inf = 0 times the row: zeros, and NaN at the infinity itself
    assert torch.isnan(y[2, 9]) and not y[2, :9].any() and torch.isnan(q[2, 9].float())
    # far below eps: y = 1e-27, still a scale and values of full size
    assert bool((q[3].float() == 448).all()) and 0 < float(s[3]) < 1e-28
    check_fp8(q[4:], s[4:], formula(x[4:], None, None, 1e-6)[0])


def test_no_rows_and_other_streams():
    w = torch.ones(64, device="cuda")
    assert rms_norm(torch.empty(0, 64, device="cuda"), w).shape == (0, 64)
    q, s = rms_norm_fp8(torch.empty(0, 64, device="cuda"), w)
    assert q.shape == (0, 64) and s.shape == (0,)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        x = torch.randn(512, 4096, device="cuda") * 3
        y = rms_norm(x, None)
    side.synchronize()
    check(y, formula(x, None, None, 1e-6)[0], torch.float32)


def test_repeats_bit_for_bit():
    x, w, r = inputs(257, 5120, torch.bfloat16, True)
    a, b = (rms_norm_fp8(x, w, residual=r) for _ in range(2))
    assert all(torch.equal(u.view(torch.uint8), v.view(torch.uint8)) for u, v in zip(a, b))


def test_refusals():
    x, w, r = inputs(4, 64, torch.bfloat16, True)
    for bad in (dict(weight=w[:32]), dict(weight=w.float()), dict(residual=r[:2]),
                dict(residual=r.float()), dict(residual=r, residual_out=r.float()),
                dict(out=torch.empty(4, 63, device="cuda", dtype=torch.bfloat16))):
        kw = dict(weight=w)
        kw.update(bad)
        with pytest.raises(ValueError):
            rms_norm(x, **kw)
    with pytest.raises(ValueError):
        rms_norm(x.cpu(), w.cpu())
    with pytest.raises(TypeError):
        rms_norm(x.double(), w.double())
    with pytest.raises(ValueError):
        rms_norm_fp8(x[:, :0], w[:0])


@pytest.mark.parametrize("rows,n", [(6000, 120), (1500, 5120), (3000, 1031), (700, 16000), (200, 20000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_blocks_that_walk_rows(rows, n, dtype):
    """More rows than blocks fit: bit for bit what calls of a few rows give."""
    x, w, r = inputs(rows, n, dtype, True, 5)
    y, s = rms_norm(x, w, 1e-6, residual=r)
    q, sc, s8 = rms_norm_fp8(x, w, 1e-6, residual=r)
    for i in range(0, rows, 100):
        e = slice(i, i + 100)
        y1, s1 = rms_norm(x[e], w, 1e-6, residual=r[e])
        q1, sc1, s81 = rms_norm_fp8(x[e], w, 1e-6, residual=r[e])
        assert torch.equal(y[e], y1) and torch.equal(s[e], s1) and torch.equal(s8[e], s81)
        assert torch.equal(q[e].view(torch.uint8), q1.view(torch.uint8))
        assert torch.equal(sc[e], sc1)
    out, kept = rms_norm(x, w, 1e-6, residual=r, out=x, residual_out=r)  # the stream in place
    assert out is x and kept is r and torch.equal(out, y) and torch.equal(kept, s)
