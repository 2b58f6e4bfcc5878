"""Attention's schedules beyond the small calls: warps on several heads at the same tokens (calls
of many steps), a head for every warp, head blocks that are not full, the copies of pages that
are no multiple of 8, and batches that are cut into several launches.  Against the formula in 64
bits, with the bounds of the other attention tests."""
import pytest
import torch

from test_paged_kv_gpu import BF, E4M3, HF, check_attend, gen, make_cache, make_table, run

pytestmark = pytest.mark.gpu


def heads_wide(vheads, warps):
    best, most = 1, 0.0
    for h in range(1, min(vheads, warps, 8) + 1):
        busy = vheads / (-(-vheads // h) * h) * (warps // h * h) / warps
        busy *= 1.0 if h >= 4 else 0.9 if h >= 2 else 0.8
        if busy >= most:
            best, most = h, busy
    return best


def visible_granules(n, window, sinks):
    if not window or n <= window:
        return -(-n // 8)
    first = n - window
    return -(-min(sinks, first) // 8) + -(-n // 8) - first // 8


def assert_wide(lens, hq, hkv, D, width, window=None, sinks=0):
    """The call counts as large, with `width` warps abreast (16-bit caches)."""
    group = hq // hkv
    vheads = hkv * -(-group // 16)
    dp = 64 if D <= 64 else 128 if D <= 128 else 256
    warps, tokens = (4 if dp > 128 else 12), (32 if dp == 64 else 16)
    assert heads_wide(vheads, warps) == width
    step = warps // width * tokens // 8
    steps = sum(-(-visible_granules(n, window, sinks) // step) for n in lens) * -(-vheads // width)
    assert steps >= 8 * torch.cuda.get_device_properties(0).multi_processor_count


RAGGED = [4000, 1, 0, 2999, 17, 3001, 48, 5000, 0, 96, 2048, 4095, 700, 33, 0, 3500, 2500, 4500]


@pytest.mark.parametrize("hq,hkv,D,width", [
    (16, 8, 128, 4), (14, 7, 128, 4), (10, 5, 128, 5), (24, 12, 64, 6), (9, 9, 128, 3),
    (10, 10, 80, 2), (40, 2, 128, 4), (11, 11, 96, 6), (21, 21, 64, 3)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_warps_on_several_heads(hq, hkv, D, width, dtype):
    lens = RAGGED * (3 if hkv < 6 else 2)
    assert_wide(lens, hq, hkv, D, width)
    run(lens, hq, hkv, D, 16, dtype, seed=hkv)


@pytest.mark.parametrize("hq,hkv,D,width", [(8, 4, 256, 4), (14, 7, 256, 4), (16, 8, 192, 4),
                                            (80, 2, 144, 2), (132, 4, 256, 4), (6, 6, 256, 2)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_a_head_for_every_warp(hq, hkv, D, width, dtype):
    # four warps a block: four heads wide leave each warp a head of its own
    assert_wide(RAGGED, hq, hkv, D, width)
    run(RAGGED, hq, hkv, D, 16, dtype, seed=hkv)


@pytest.mark.parametrize("hq,hkv,D,width,window,sinks", [
    (12, 12, 64, 6, 1024, 4), (14, 7, 128, 4, 1000, 0), (8, 8, 256, 4, 513, 20),
    (10, 5, 128, 5, 2047, 300)])
def test_windows_of_large_calls(hq, hkv, D, width, window, sinks):
    lens = RAGGED * 4
    assert_wide(lens, hq, hkv, D, width, window, sinks)
    run(lens, hq, hkv, D, 16, HF, window=window, sinks=sinks, seed=D)


@pytest.mark.parametrize("hq,hkv,D,width", [(16, 8, 128, 4), (8, 4, 256, 4)])
def test_large_calls_repeat_and_do_not_mind_missing_pages(hq, hkv, D, width):
    assert_wide(RAGGED, hq, hkv, D, width)
    o, q, cache, table, ln = run(RAGGED, hq, hkv, D, 16)
    assert all(torch.equal(o, cache.attend(q, table, ln)) for _ in range(5))
    table = table.clone()
    table[0, 7:60], table[3, ::5], table[5] = -1, cache.pages, -3
    check_attend(cache.attend(q, table, ln), q, cache, table, RAGGED)


@pytest.mark.parametrize("page", [1, 12, 20])
@pytest.mark.parametrize("hq,hkv,D", [(4, 2, 80), (6, 2, 128), (8, 2, 256), (2, 2, 16)])
@pytest.mark.parametrize("dtype,cdt", [(HF, HF), (BF, BF), (HF, E4M3)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (50, 3)])
def test_pages_that_are_no_multiple_of_8(page, hq, hkv, D, dtype, cdt, window, sinks):
    run([0, 1, 7, 8, 9, 100, 333, 640], hq, hkv, D, page, dtype, cdt, window=window, sinks=sinks,
        layout="head")


def test_large_call_over_pages_that_are_no_multiple_of_8():
    assert_wide(RAGGED, 16, 8, 128, 4)
    run(RAGGED, 16, 8, 128, 12)
    assert_wide(RAGGED, 8, 4, 256, 4)
    run(RAGGED, 8, 4, 256, 20, HF, window=1500, sinks=9)


def test_batch_of_more_items_than_a_launch_takes():
    # 2^18 (sequence, head) items of a launch: 4096 sequences of 64 heads, and the rest
    B, heads = 9001, 64
    cache = make_cache(B, 8, heads, 16, BF)
    order = torch.randperm(B, generator=torch.Generator().manual_seed(1))
    table = order.to(torch.int32)[:, None].cuda()
    lens = torch.randint(0, 2, (B,), generator=gen(2), device="cuda").to(torch.int32)
    q = torch.randn(B, heads, 16, generator=gen(3), device="cuda").to(BF)
    o = cache.attend(q, table, lens)
    want = cache.v[order.cuda(), 0] * lens[:, None, None].to(BF)  # a token alone: its values
    assert torch.equal(o, want)


def test_tables_of_more_steps_than_a_launch_takes():
    # 2^24 tokens a sequence by the table, 64 heads: 15 sequences of a launch
    B, heads, page = 40, 64, 1 << 20
    cache = make_cache(1, page, heads, 16, E4M3)
    table = torch.full((B, 16), -1, dtype=torch.int32, device="cuda")
    table[:, 0] = 0
    lens = [1 + 37 * b for b in range(B - 1)] + [1 << 24]
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn(B, heads, 16, generator=gen(4), device="cuda").to(BF)
    check_attend(cache.attend(q, table, ln), q, cache, table, lens)  # one page is there


@pytest.mark.parametrize("hq,hkv,D,cdt", [(8, 2, 128, BF), (8, 4, 256, BF), (16, 16, 64, E4M3)])
@pytest.mark.parametrize("live", [(0, 1, 299), (150,), (149, 296, 297), ()])
def test_padding_among_the_sequences(hq, hkv, D, cdt, live):
    lens = [0] * 300
    for i, b in enumerate(live):
        lens[b] = 40 + 333 * i
    cache = make_cache(80, 16, hkv, D, cdt)
    table = make_table(lens, 16, 80, width=45)
    q = torch.randn(300, hq, D, generator=gen(5), device="cuda").to(BF)
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = torch.full_like(q, float("nan"))
    cache.attend(q, table, ln, out=out)
    check_attend(out, q, cache, table, lens)
