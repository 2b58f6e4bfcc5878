"""The paged cache: append (RoPE, 16-bit and e4m3 storage) and attention of one new token per
sequence, against their formulas in 64 bits.

Bounds.  Append: k and q are two f32 products and a sum, 2^-22 of |x0| + |x1|, then the output's
rounding; v in 16 bits is copied exactly; e4m3: 2^-4 relative, 2^-10 where subnormal.
Attention, with W = sum p |v| / sum p per output: the weights p count with 11 bits or more
(f16: 2^-11; bf16 by two MMAs: 2^-16), the scores and exponentials add less than 2^-12 at these
sizes, so |err| <= W 2^-10 + the output's rounding (2^-8 |o| bf16, 2^-11 |o| + 2^-25 f16)."""
import math

import pytest
import torch

from sketchpad_b200 import PagedKVCache, SketchpadError

pytestmark = pytest.mark.gpu
ROUND = {torch.bfloat16: (2.0 ** -8, 0.0), torch.float16: (2.0 ** -11, 2.0 ** -25)}
E4M3 = torch.float8_e4m3fn
BF, HF = torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make_cache(pages, page, hkv, D, dtype, seed=0, layout="slot"):
    g = gen(seed + 1)
    shape = (pages, page, hkv, D) if layout == "slot" else (pages, hkv, page, D)
    ks = vs = None
    if dtype == E4M3:
        ks = 0.005 + 0.02 * torch.rand(hkv, generator=g, device="cuda")
        vs = 0.005 + 0.02 * torch.rand(hkv, generator=g, device="cuda")
    t = []
    for _ in range(2):
        v = torch.randn(shape, generator=g, device="cuda")
        v = (v * 60).clamp(-448, 448).to(E4M3) if dtype == E4M3 else v.to(dtype)
        t.append(v if layout == "slot" else v.transpose(1, 2))
    return PagedKVCache(t[0], t[1], ks, vs)


def make_table(lens, page, pages, seed=0, width=None):
    need = [-(-n // page) for n in lens]
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    assert sum(need) <= pages
    t = torch.full((len(lens), width or max(max(need), 1)), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        t[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    return t.cuda()


def dense(cache, table, b, toks):
    p = table[b].long()[toks // cache.page_size]
    u8 = lambda t: t.view(torch.uint8) if t.dtype == E4M3 else t  # noqa: E731
    k = u8(cache.k)[p, toks % cache.page_size].view(cache.k.dtype).double()
    v = u8(cache.v)[p, toks % cache.page_size].view(cache.v.dtype).double()
    if cache.k_scale is not None:
        k, v = k * cache.k_scale.double()[:, None], v * cache.v_scale.double()[:, None]
    return k.transpose(0, 1), v.transpose(0, 1)  # [hkv, n, D]


def check_attend(o, q, cache, table, lens, window=None, sinks=0, scale=None):
    B, hq, D = q.shape
    scale = scale or 1 / math.sqrt(D)
    for b, n in enumerate(lens):
        n = max(0, min(n, table.shape[1] * cache.page_size))
        toks = torch.arange(n, device="cuda")
        if window:
            toks = toks[(toks >= n - window) | (toks < sinks)]
        if n:
            page = table[b].long()[toks // cache.page_size]
            toks = toks[(page >= 0) & (page < cache.pages)]
        if toks.numel() == 0:
            assert not o[b].any()
            continue
        k, v = dense(cache, table, b, toks)
        qq = q[b].double().reshape(cache.kv_heads, -1, D)
        p = torch.softmax(qq @ k.transpose(1, 2) * scale, -1)
        ref, w = (p @ v).reshape(hq, D), (p @ v.abs()).reshape(hq, D)
        rel, absolute = ROUND[q.dtype]
        bound = w * 2.0 ** -10 + ref.abs() * rel + absolute
        err = (o[b].double() - ref).abs()
        assert bool((err <= bound).all()), (b, n, float((err / bound).max()))


def run(lens, hq, hkv, D, page, dtype=BF, cdt=None, seed=0, layout="slot", **kw):
    total = sum(-(-n // page) for n in lens) + 2
    cache = make_cache(total, page, hkv, D, cdt or dtype, seed, layout)
    table = make_table(lens, page, total, seed)
    q = torch.randn(len(lens), hq, D, generator=gen(seed), device="cuda").to(dtype)
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    o = cache.attend(q, table, ln, **kw)
    assert o.shape == q.shape and o.dtype == q.dtype
    check_attend(o, q, cache, table, lens, **kw)
    return o, q, cache, table, ln


@pytest.mark.parametrize("hq,hkv", [(8, 8), (8, 2), (5, 1), (14, 2), (16, 1), (40, 2), (33, 1)])
@pytest.mark.parametrize("dtype,cdt", [(BF, BF), (HF, HF), (BF, E4M3), (HF, E4M3)])
def test_heads_and_types(hq, hkv, dtype, cdt):
    run([1, 17, 300, 0, 129], hq, hkv, 128, 16, dtype, cdt)


@pytest.mark.parametrize("D", [16, 32, 48, 64, 80, 96, 112, 128, 144, 192, 256])
@pytest.mark.parametrize("dtype,cdt", [(BF, BF), (HF, HF), (BF, E4M3)])
def test_head_dims(D, dtype, cdt):
    run([1, 64, 333], 6, 2, D, 16, dtype, cdt, seed=D)


@pytest.mark.parametrize("page", [1, 3, 7, 16, 24, 64, 100, 256])
@pytest.mark.parametrize("cdt", [BF, E4M3])
def test_page_sizes_and_lengths(page, cdt):
    run([0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 500], 4, 2, 64, page, BF, cdt)


@pytest.mark.parametrize("lens", [[20011], [1] * 300, [9000] + [3] * 40 + [0] * 9 + [5000],
                                  [0] * 5, [4097] * 3])
@pytest.mark.parametrize("cdt", [BF, E4M3])
def test_ragged_batches(lens, cdt):
    run(lens, 8, 2, 128, 32, BF, cdt)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (100, 0), (100, 7), (128, 200),
                                          (5000, 4), (1000, 64)])
@pytest.mark.parametrize("cdt", [HF, E4M3])
def test_window_and_sinks(window, sinks, cdt):
    run([0, 1, 5, 16, 99, 100, 101, 110, 128, 1500, 3000], 4, 4, 64, 16, HF, cdt, window=window,
        sinks=sinks)


def test_orders_and_strides():
    run([700, 33], 8, 2, 128, 16, layout="head")
    run([700, 33], 8, 2, 64, 16, BF, E4M3, layout="head")
    # q as a view of a projection's output, heads 4-byte aligned only, and a table view
    cache = make_cache(40, 16, 2, 64, BF)
    table = torch.cat((make_table([300, 200], 16, 40), make_table([8, 8], 16, 40)), 1)[:, :19]
    lens = [300, 200]
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    qkv = torch.randn(2, 12, 64, device="cuda").to(BF)
    check_attend(cache.attend(qkv[:, 3:11], table, ln), qkv[:, 3:11], cache, table, lens)
    odd = torch.randn(2, 8 * 64 + 1, device="cuda").to(BF)[:, 1:].reshape(2, 8, 64)
    wide = torch.randn(2, 8, 66, device="cuda").to(BF)[..., 1:65]
    for q in (odd, wide):
        check_attend(cache.attend(q, table, ln, scale=0.3), q, cache, table, lens, scale=0.3)


def test_slots_outside_the_lengths_hold_anything():
    o, q, cache, table, ln = run([37, 0, 90], 4, 2, 128, 16)
    used = torch.zeros(cache.pages, 16, dtype=torch.bool, device="cuda")
    for b, n in enumerate([37, 0, 90]):
        t = torch.arange(n, device="cuda")
        used[table[b].long()[t // 16], t % 16] = True
    cache.k[~used] = float("nan")
    cache.v[~used] = float("inf")
    assert torch.equal(cache.attend(q, table, ln), o)


def test_pages_that_are_not_there():
    lens = [200, 64, 48]
    cache = make_cache(30, 16, 2, 64, BF)
    table = make_table(lens, 16, 30)
    table[0, 2], table[0, 7], table[0, 12] = -1, 30, 2 ** 31 - 1
    table[1, :] = -5
    q = torch.randn(3, 4, 64, device="cuda").to(BF)
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    check_attend(cache.attend(q, table, ln), q, cache, table, lens)
    # lengths beyond the table, and negative ones
    lens = [5000, -3, 2 ** 31 - 1]
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    check_attend(cache.attend(q, table, ln), q, cache, table, lens)


def test_offsets_beyond_32_bits():
    base = torch.empty(2 ** 31 + 2 ** 21, dtype=HF, device="cuda")
    k = base.as_strided((3, 16, 2, 64), (2 ** 30, 128, 64, 1))
    v = base[2 ** 20:].as_strided((3, 16, 2, 64), (2 ** 30, 128, 64, 1))
    k.normal_()
    v.normal_()
    cache = PagedKVCache(k, v)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 4, 64, device="cuda").to(HF)
    ln = torch.tensor([41], dtype=torch.int32, device="cuda")
    check_attend(cache.attend(q, table, ln), q, cache, table, [41])
    new = torch.randn(1, 2, 64, device="cuda").to(HF)
    one = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache.append(new, -new, table, one, one + 5)
    assert torch.equal(cache.k[2, 5], new[0]) and torch.equal(cache.v[2, 5], -new[0])


def test_large_scores_and_special_values():
    lens = [300, 300, 300, 300]
    cache = make_cache(80, 16, 1, 64, BF)
    table = make_table(lens, 16, 80)
    q = torch.randn(4, 4, 64, device="cuda").to(BF)
    q[1] *= 1e4          # one key takes everything
    q[2] = 0             # the plain mean
    q[3, 0] = float("nan")
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    o = cache.attend(q, table, ln)
    assert torch.isnan(o[3, 0]).all() and torch.isfinite(o[:3].float()).all()
    k, v = dense(cache, table, 1, torch.arange(300, device="cuda"))
    best = (q[1].double() @ k[0].t()).argmax(-1)
    assert torch.equal(o[1].double(), v[0][best])
    check_attend(o[2:3], q[2:3], cache, table[2:3], [300])
    # e4m3 caches take queries beyond f16's range, and very small ones
    cache = make_cache(80, 16, 1, 64, E4M3)
    for f in (1e30, 1e-30):
        q = (torch.randn(4, 4, 64, device="cuda") * f).to(BF)
        o = cache.attend(q, table, ln, scale=0.125 / f)
        check_attend(o, q, cache, table, lens, scale=0.125 / f)


def test_repeats_streams_and_workspaces():
    o, q, cache, table, ln = run([5000, 1, 777, 64], 8, 2, 128, 16)
    assert all(torch.equal(o, cache.attend(q, table, ln)) for _ in range(10))
    # calls of other sizes on the same workspace, between
    for lens in ([100] * 4, [0, 0, 1, 0], [5000, 1, 777, 64]):
        l2 = torch.tensor(lens, dtype=torch.int32, device="cuda")
        check_attend(cache.attend(q, table, l2), q, cache, table, lens)
    many = table[:1].expand(200, -1).contiguous()
    qm = torch.randn(200, 8, 128, device="cuda").to(BF)
    lm = torch.full((200,), 700, dtype=torch.int32, device="cuda")
    check_attend(cache.attend(qm, many, lm), qm, cache, many, [700] * 200)
    assert torch.equal(o, cache.attend(q, table, ln))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(cache.attend(q, table, ln))
    torch.cuda.synchronize()
    assert all(torch.equal(o, x) for x in outs)
    w = cache.new_workspace(8)
    assert torch.equal(o, cache.attend(q, table, ln, workspace=w))
    assert not w[:1 << 18].any()


def test_attend_in_a_graph():
    o, q, cache, table, ln = run([2000, 5], 8, 2, 128, 16)
    w, out = cache.new_workspace(8), torch.zeros_like(q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.attend(q, table, ln, out=out, workspace=w)
    for lens in ([2000, 5], [1, 80], [0, 2000]):
        ln.copy_(torch.tensor(lens, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        n = [min(x, y) for x, y in zip(lens, [2000, 16])]
        check_attend(out, q, cache, table, [lens[0], lens[1]])
        assert n is not None


# ------------------------------------------------------------------------------------ append
def rope_table(n, D):
    ang = torch.arange(n)[:, None] * torch.exp(torch.arange(D // 2) * (-2 * math.log(1e4) / D))
    return torch.stack((ang.cos(), ang.sin()), -1).float().contiguous().cuda()


def rotate(x, cs):
    a, b = x[..., 0::2].double(), x[..., 1::2].double()
    c, s = cs[:, None, :, 0].double(), cs[:, None, :, 1].double()
    size = (a.abs() + b.abs()).repeat_interleave(2, -1)
    return torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2), size


def check_round(got, ref, size, dtype):
    err = (got.double() - ref).abs()
    if dtype == E4M3:
        bound = torch.maximum(ref.abs() * 2.0 ** -4, torch.full_like(ref, 2.0 ** -10))
        bound = bound + size * 2.0 ** -21
        ref = ref.clamp(-448, 448)
        err = (got.double() - ref).abs()
    else:
        bound = ref.abs() * ROUND[dtype][0] + ROUND[dtype][1] + size * 2.0 ** -22
    assert bool((err <= bound).all()), float((err - bound).max())


@pytest.mark.parametrize("T", [1, 3, 130])
@pytest.mark.parametrize("hq,hkv,D", [(8, 2, 128), (3, 3, 64), (5, 1, 16), (4, 2, 80), (16, 1, 256),
                                      (40, 8, 128)])
@pytest.mark.parametrize("dtype,cdt", [(BF, BF), (HF, HF), (BF, E4M3), (HF, E4M3)])
@pytest.mark.parametrize("rope", [False, True])
def test_append(T, hq, hkv, D, dtype, cdt, rope):
    B, page = 3, 16
    cache = make_cache(40, page, hkv, D, cdt, layout="head" if T == 3 else "slot")
    k0, v0 = cache.k.clone(), cache.v.clone()
    table = make_table([150, 100, 60], page, 40)
    g = gen(T)
    seq = torch.arange(T, device="cuda").to(torch.int32) % B
    pos = 5 + torch.arange(T, device="cuda").to(torch.int32) // B
    qkv = (torch.randn(T, hq + 2 * hkv, D, generator=g, device="cuda") * 2).to(dtype)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    cs = rope_table(64, D) if rope else None
    out = cache.append(k, v, table, seq, pos, q=q, rope=cs)
    at = table[seq.long(), pos.long() // page].long(), pos.long() % page
    u8 = lambda t: t.view(torch.uint8) if t.dtype == E4M3 else t  # noqa: E731
    ident = lambda x: (x.double(), torch.zeros_like(x.double()))  # noqa: E731
    turn = (lambda x: rotate(x, cs[pos.long()])) if rope else ident
    ref, size = turn(q)
    check_round(out, ref, size, dtype)
    for new, now, before, s, (ref, size) in ((k, cache.k, k0, cache.k_scale, turn(k)),
                                             (v, cache.v, v0, cache.v_scale, ident(v))):
        if s is not None:
            ref, size = (t / s.double()[:, None] for t in (ref, size))
        got = u8(now)[at].view(now.dtype)
        check_round(got, ref, size, cdt)
        if cdt != E4M3 and not (rope and new is k):
            assert torch.equal(got, new)
        untouched = torch.ones(now.shape[:2], dtype=torch.bool, device="cuda")
        untouched[at] = False
        assert torch.equal(u8(now)[untouched], u8(before)[untouched])


@pytest.mark.parametrize("hq,hkv,D", [(40, 8, 128), (14, 2, 256), (56, 8, 256), (5, 1, 80),
                                      (0, 3, 64)])
@pytest.mark.parametrize("cdt", [BF, E4M3])
def test_append_long_calls(hq, hkv, D, cdt):
    """Many tokens take fewer threads each: bit for bit what the same tokens give in short calls
    (which test_append compares with 64 bits)."""
    T, B, page = 1531, 3, 16
    ca, cb = (make_cache(110, page, hkv, D, cdt) for _ in range(2))
    table = make_table([T // B + 30] * B, page, 110)
    seq = torch.arange(T, device="cuda").to(torch.int32) % B
    pos = 7 + torch.arange(T, device="cuda").to(torch.int32) // B
    pos[100] = -1
    qkv = torch.randn(T, hq + 2 * hkv, D, generator=gen(hq), device="cuda").to(BF)
    q = qkv[:, :hq].contiguous() if hq else None
    k, v = qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    cs = rope_table(T, D)
    want = []
    for i in range(0, T, 500):
        e = slice(i, i + 500)
        want.append(ca.append(k[e], v[e], table, seq[e], pos[e], q=q[e] if hq else None, rope=cs))
    got = cb.append(k, v, table, seq, pos, q=q, rope=cs)
    for x, y in ((ca.k, cb.k), (ca.v, cb.v)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    if hq:
        assert torch.equal(torch.cat(want), got) and not got[100].any()
        assert cb.append(k, v, table, seq, pos, q=q, rope=cs, q_out=q) is q  # in place
        assert torch.equal(q, got)
    else:
        assert got is None


def test_append_padding_and_missing_pages():
    cache = make_cache(10, 8, 2, 64, BF)
    k0 = cache.k.clone()
    table = make_table([40, 16], 8, 10, width=5)
    table[0, 1], table[0, 2] = -1, 10
    cs = rope_table(30, 64)
    #           ok, page -1, page 10, negative, past the table, past rope, bad sequences, ok
    seq = torch.tensor([0, 0, 0, 0, 1, 0, -1, 2, 1], dtype=torch.int32, device="cuda")
    pos = torch.tensor([3, 9, 17, -1, 60, 31, 0, 0, 12], dtype=torch.int32, device="cuda")
    q = torch.randn(9, 4, 64, device="cuda").to(BF)
    k = torch.randn(9, 2, 64, device="cuda").to(BF)
    out = cache.append(k, k, table, seq, pos, q=q, rope=cs)
    live = [0, 8]
    assert not out[1:8].any()
    ref, size = rotate(q[live], cs[pos[live].long()])
    check_round(out[live], ref, size, BF)
    mask = torch.ones(10, 8, dtype=torch.bool, device="cuda")
    mask[table[0, 0].long(), 3] = mask[table[1, 1].long(), 4] = False
    assert torch.equal(cache.k[mask], k0[mask])
    assert torch.equal(cache.v[table[1, 1].long(), 4], k[8])
    assert cache.append(k[:0], k[:0], table, seq[:0], pos[:0]) is None
    # q rotated in place
    qc = q.clone()
    assert cache.append(k, k, table, seq, pos, q=qc, rope=cs, q_out=qc) is qc
    assert torch.equal(qc, out)


def test_refusals():
    cache = make_cache(8, 16, 2, 64, BF)
    table = make_table([40, 16], 16, 8)
    ln = torch.tensor([40, 16], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 4, 64, device="cuda").to(BF)
    k = q[:, :2]
    for bad in (lambda: cache.attend(q[:, :3], table, ln), lambda: cache.attend(q.half(), table, ln),
                lambda: cache.attend(q[..., :32], table, ln), lambda: cache.attend(q, table, ln[:1]),
                lambda: cache.attend(q, table.long(), ln), lambda: cache.attend(q, table, ln.long()),
                lambda: cache.attend(q, table, ln, window=0),
                lambda: cache.attend(q, table, ln, sinks=-1),
                lambda: cache.attend(q, table, ln, out=q.float()),
                lambda: cache.attend(q.cpu(), table, ln),
                lambda: cache.append(k, k, table, ln, ln[:1]),
                lambda: cache.append(k, k.half(), table, ln, ln),
                lambda: cache.append(k[..., :32], k[..., :32], table, ln, ln),
                lambda: cache.append(k, k, table, ln, ln, rope=rope_table(4, 32)),
                lambda: cache.append(k, k, table, ln, ln, q_out=q),
                lambda: PagedKVCache(cache.k, cache.v[:4]),
                lambda: PagedKVCache(cache.k, cache.v, ln.float(), ln.float()),
                lambda: PagedKVCache(cache.k.to(E4M3), cache.v.to(E4M3))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        PagedKVCache(cache.k.float(), cache.v.float())
    with pytest.raises(SketchpadError):  # too small a workspace
        cache.attend(q, table, ln, workspace=torch.zeros(4, device="cuda", dtype=torch.int32))
    for D in (24, 264):  # head dims outside the multiples of 16 up to 256
        t = torch.zeros(4, 16, 2, D, device="cuda", dtype=BF)
        with pytest.raises(SketchpadError):
            PagedKVCache(t, t).attend(torch.zeros(2, 4, D, device="cuda", dtype=BF), table, ln)
    t = torch.zeros(4, 16, 2, 68, device="cuda", dtype=BF)[..., :64]  # rows off 16 bytes
    with pytest.raises(SketchpadError):
        PagedKVCache(t, t).attend(q, table, ln)
