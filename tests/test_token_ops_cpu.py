"""Host side of the token operators without a GPU: argument errors of the C entries, sizes, the
cache handle, and what the Python layer refuses."""
import ctypes

import pytest
import torch

from sketchpad_b200 import Int4Linear, PagedKVCache, _lib, rms_norm, rms_norm_fp8
from sketchpad_b200.decoder import DecoderConfig, rope_table

L = _lib.load()
P = lambda a: ctypes.c_void_p(a)  # noqa: E731  an address that is checked but never read
i4 = _lib.i64_array


def test_rms_norm_arguments():
    ok = (P(256), 64, None, 64, P(256), P(512), None, 4, 64, 1e-6, 2, None)

    def call(**kw):
        names = ("x", "xs", "res", "rs", "w", "y", "ro", "rows", "n", "eps", "dtype", "stream")
        a = dict(zip(names, ok))
        a.update(kw)
        return L.sp_rms_norm(*[a[k] for k in names])

    assert call(x=None) == -1 and call(y=None) == -1
    assert call(n=0) == -1 and call(rows=-1) == -1
    assert call(xs=63) == -2 and call(res=P(256), rs=8) == -2
    assert call(dtype=3) == -3 and call(dtype=9) == -3
    assert call(n=2 ** 31) == -2
    assert call(rows=0) == 0 and call(rows=0, x=None, y=None) == 0
    assert L.sp_rms_norm_fp8(P(256), 64, None, 64, None, P(512), None, None, 4, 64, 1e-6, 2,
                             None) == -1  # no scale


def test_int4_sizes_and_arguments():
    sizes = i4((0, 0, 0, 0))
    # tiles of 32 outputs x 128 inputs: 2 KB, 32 scales of 2 bytes and 32 zeros per group of it
    for N, K, group, tiles, chunks, gpc in ((1, 32, 32, 1, 1, 4), (33, 192, 64, 2, 2, 2),
                                            (64, 4096, 256, 2, 32, 1)):
        assert L.sp_int4_packed_bytes(N, K, group, sizes) == 0
        assert list(sizes)[:3] == [tiles * chunks * b for b in (2048, 64 * gpc, 32 * gpc)]
    for N, K, group, rc in ((0, 32, 32, -1), (8, 0, 32, -1), (8, 64, 0, -1), (8, 96, 96, -2),
                            (8, 48, 32, -2), (8, 128, 16, -2), (2 ** 31, 32, 32, -2)):
        assert L.sp_int4_packed_bytes(N, K, group, sizes) == rc
    assert L.sp_int4_packed_bytes(8, 32, 32, None) == -1
    # the workspace does not shrink with M up to 32, and stays there
    need = [L.sp_int4_linear_workspace_size(m, 5120, 13824, 32) for m in (8, 16, 32, 33, 1000)]
    assert all(n >= 256 * 1024 for n in need) and need[2] == need[3] == need[4]
    assert L.sp_int4_linear_workspace_size(0, 8, 32, 32) == 0

    def linear(x=P(256), stride=256, xd=2, xs=None, q=P(256), s=P(256), sd=1, y=P(256), M=4, N=16,
               K=256, group=64, out=2):
        return L.sp_int4_linear(x, stride, xd, xs, q, s, None, sd, None, y, M, N, K, group, out,
                                None, 0, None)

    assert linear(x=None) == -1 and linear(q=None) == -1 and linear(y=None) == -1
    assert linear(M=-1) == -1 and linear(xs=P(256)) == -1 and linear(xd=3) == -1
    assert linear(xd=0) == -3 and linear(sd=0) == -3 and linear(out=3) == -3
    assert linear(stride=255) == -2 and linear(N=2 ** 22) == -2
    assert linear(stride=260) == -4 and linear(x=P(264)) == -4 and linear(q=P(8)) == -4
    assert linear(M=0) == 0


def make(k=P(4096), v=P(8192), ks=None, vs=None, st=(2048, 128, 64, 1), pages=4, page=16, hkv=2,
         D=64, dtype=2):
    h = ctypes.c_void_p()
    rc = L.sp_paged_cache_create(k, v, ks, vs, i4(st), i4(st), pages, page, hkv, D, dtype,
                                 ctypes.byref(h))
    return rc, h


def test_paged_cache_handle():
    rc, h = make()
    assert rc == 0 and h.value
    assert L.sp_paged_cache_destroy(h) == 0 and L.sp_paged_cache_destroy(None) == 0
    for bad, want in ((dict(k=None), -1), (dict(pages=0), -1), (dict(page=0), -1),
                      (dict(D=24), -2), (dict(D=272), -2), (dict(dtype=0), -3),
                      (dict(dtype=3), -1), (dict(st=(2048, 128, 68, 1)), -4),
                      (dict(st=(2048, 128, 64, 2)), -4), (dict(k=P(4100)), -4),
                      (dict(pages=2 ** 31), -2)):
        rc, h = make(**bad)
        assert rc == want and not h.value, bad


def test_paged_calls_check_their_arguments():
    rc, h = make()
    assert rc == 0

    def attend(h=h, q=P(256), qs=256, qh=64, table=P(256), cols=8, ts=8, lens=P(256), out=P(256),
               B=2, hq=4, window=0, sinks=0, dtype=2, ws=None, wb=0):
        return L.sp_paged_attention(h, q, qs, qh, table, cols, ts, lens, out, B, hq, window, sinks,
                                    0.0, dtype, ws, wb, None)

    assert attend(h=None) == -1 and attend(q=None) == -1 and attend(lens=None) == -1
    assert attend(B=-1) == -1 and attend(hq=0) == -1 and attend(table=None) == -1
    assert attend(cols=0) == -1 and attend(window=-1) == -1 and attend(sinks=-1) == -1
    assert attend(hq=3) == -2 and attend(ts=7) == -2 and attend(cols=2 ** 28, ts=2 ** 28) == -2
    assert attend(dtype=1) == -3 and attend(dtype=0) == -3
    assert attend(qs=255) == -4 and attend(q=P(258)) == -4 and attend(out=P(264)) == -4
    assert attend(B=0) == 0
    assert L.sp_paged_attention_workspace_size(4, 2, 64) > 2 ** 20
    assert L.sp_paged_attention_workspace_size(3, 2, 64) == 0

    def append(h=h, q=P(256), k=P(256), qo=P(256), hq=4, kt=128, rows=2, cols=8, rope=None, rr=0,
               dtype=2, T=3, seq=P(256)):
        return L.sp_paged_kv_append(h, q, k, P(256), qo, 256, 64, kt, 64, 128, 64, T, hq, P(256),
                                    rows, cols, cols, seq, P(256), rope, rr, dtype, None)

    assert append(h=None) == -1 and append(k=None) == -1 and append(seq=None) == -1
    assert append(qo=None) == -1 and append(q=None) == -1 and append(hq=0) == -1
    assert append(T=-1) == -1 and append(rope=P(256), rr=0) == -1 and append(rows=-1) == -1
    assert append(dtype=1) == -3 and append(kt=132) == -4 and append(k=P(264)) == -4
    assert append(T=0) == 0
    assert L.sp_paged_cache_destroy(h) == 0


def test_python_layer_refuses_host_tensors():
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    for f in (rms_norm, rms_norm_fp8):
        with pytest.raises(ValueError):
            f(x, None)
    with pytest.raises(ValueError):
        Int4Linear(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(2, 4, dtype=torch.float16),
                   group_size=32)
    with pytest.raises(ValueError):
        PagedKVCache(torch.zeros(2, 16, 2, 64), torch.zeros(2, 16, 2, 64))


def test_rope_table_pairs():
    c = DecoderConfig(hidden=64, intermediate=64, heads=1, kv_heads=1, head_dim=8,
                      max_positions=50)
    t = rope_table(c, "cpu").double()
    assert t.shape == (50, 4, 2) and torch.equal(t[0], torch.tensor([[1.0, 0.0]] * 4).double())
    for pos in (1, 49):
        for i in range(4):
            a = pos * 10000.0 ** (-2 * i / 8)
            want = torch.tensor([a, a - torch.pi / 2], dtype=torch.float64).cos()
            assert torch.allclose(t[pos, i], want, atol=2.0 ** -24)


@pytest.mark.parametrize("N,K,group", [(144, 4096, 32), (32, 1408, 128), (5120, 13824, 32),
                                       (235, 17472, 64), (20832, 4864, 128)])
def test_int4_workspace_serves_any_number_of_rows(N, K, group):
    # a call beyond 32 rows runs the rest as a call of its own
    need = [L.sp_int4_linear_workspace_size(m, N, K, group) for m in range(1, 70)]
    assert need == sorted(need) and len(set(need[31:])) == 1
