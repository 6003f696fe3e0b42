"""CPU checks of the serving calls: bad arguments are refused before a device
is touched, by the C ABI and by the binding, and the plain 64-bit forms the GPU
tests compare with agree with each other."""
import ctypes
import math

import pytest
import torch

import kerr_attn
import serve_ref

P = ctypes.c_void_p


@pytest.fixture(scope="module")
def L():
    import os

    if not os.path.exists(kerr_attn.LIB_PATH):
        kerr_attn.build()
    return kerr_attn.lib()


CTX = P(0x10)  # every call below fails, or returns, before reading it
INVALID, UNSUPPORTED, MISALIGNED = (kerr_attn.KATTN_ERR_INVALID_ARGUMENT, kerr_attn.KATTN_ERR_UNSUPPORTED,
                                    kerr_attn.KATTN_ERR_MISALIGNED)


def test_fwd_packed_refusals(L):
    def call(ctx=CTX, dtype=1, q=0x1000, ldq=512, k=0x2000, v=0x3000, ldk=128, o=0x4000, ldo=512, lse=0x5000,
             cu_q=0x6000, cu_k=0x7000, S=2, Nq=9, Nk=9, H=8, Hkv=2, d=64, scale=0.125, causal=1):
        return L.kattn_fwd_packed(ctx, dtype, q, ldq, k, v, ldk, o, ldo, lse, cu_q, cu_k, S, Nq, Nk, H, Hkv, d, scale,
                                  causal, None)

    assert call(ctx=None) == INVALID
    assert call(dtype=3) == UNSUPPORTED and call(dtype=-1) == UNSUPPORTED
    assert call(d=48) == UNSUPPORTED and call(d=256, ldq=4096, ldk=4096, ldo=4096) == UNSUPPORTED
    assert call(H=9) == INVALID and call(H=0) == INVALID and call(Hkv=0) == INVALID and call(Hkv=-2) == INVALID
    assert call(S=-1) == INVALID and call(Nq=-1) == INVALID and call(Nk=-1) == INVALID
    assert call(scale=math.nan) == INVALID and call(scale=math.inf) == INVALID
    assert call(causal=2) == INVALID
    for name in ("q", "k", "v", "o", "lse", "cu_q", "cu_k"):
        assert call(**{name: None}) == INVALID, name
        assert call(**{name: 0x9002}) == MISALIGNED, name
    assert call(ldq=504) == INVALID and call(ldo=504) == INVALID and call(ldk=120) == INVALID
    assert call(ldq=516) == MISALIGNED and call(ldk=132) == MISALIGNED and call(ldo=514) == MISALIGNED
    assert call(dtype=0, ldq=518) == MISALIGNED
    assert call(ldq=1 << 40) == INVALID
    assert call(Nq=1 << 28) == INVALID and call(Nk=(1 << 31) - 1) == INVALID
    for none in (dict(S=0), dict(Nq=0)):
        assert call(q=None, k=None, v=None, o=None, lse=None, cu_q=None, cu_k=None, **none) == 0
        assert kerr_attn.last_launch_count() == 0


def table(**kw):
    t = dict(k=0x10000, v=0x20000, k_scale=0x30000, v_scale=0x40000, n_pages=4, page_size=16, n_kv_head=2, d=64, format=0)
    t.update(kw)
    return ctypes.byref(kerr_attn.KVCacheTable(*[t[n] for n, _ in kerr_attn.KVCacheTable._fields_]))


BAD_CACHES = [(dict(format=2), UNSUPPORTED), (dict(page_size=8), UNSUPPORTED), (dict(page_size=48), UNSUPPORTED),
              (dict(page_size=512), UNSUPPORTED), (dict(page_size=0), UNSUPPORTED), (dict(n_pages=-1), INVALID),
              (dict(n_kv_head=0), INVALID), (dict(d=40), UNSUPPORTED), (dict(k=None), INVALID), (dict(v=0x20008), MISALIGNED),
              (dict(k_scale=None), INVALID), (dict(v_scale=0x40002), MISALIGNED), (dict(n_kv_head=1 << 27), INVALID)]


@pytest.mark.parametrize("what", ["kattn_cache_append", "kattn_cache_read"])
def test_cache_rows_refusals(L, what):
    def call(ctx=CTX, cache=table(), dtype=1, k=0x1000, v=0x2000, ld=128, cu=0x3000, kv_len=0x4000, pages=0x5000, ldt=7,
             max_pages=7, S=2, N=9):
        return getattr(L, what)(ctx, cache, dtype, k, v, ld, cu, kv_len, pages, ldt, max_pages, S, N, None)

    assert call(ctx=None) == INVALID and call(cache=None) == INVALID
    for kw, status in BAD_CACHES:
        assert call(cache=table(**kw)) == status, kw
    assert call(dtype=7) == UNSUPPORTED
    assert call(S=-1) == INVALID and call(N=-1) == INVALID
    assert call(ld=120) == INVALID and call(ld=132) == MISALIGNED
    assert call(ldt=6) == INVALID and call(max_pages=-1) == INVALID
    assert call(ldt=1 << 27, max_pages=1 << 27) == INVALID and call(N=(1 << 31) - 1) == INVALID
    for name in ("k", "v", "cu", "kv_len", "pages"):
        assert call(**{name: None}) == INVALID, name
        assert call(**{name: 0x9002}) == MISALIGNED, name
    assert call(S=0, k=None, v=None, cu=None) == 0 and kerr_attn.last_launch_count() == 0
    assert call(N=0, k=None, v=None, cu=None) == 0


def test_fwd_cached_refusals(L):
    def call(ctx=CTX, cache=table(), dtype=2, q=0x1000, ldq=512, o=0x2000, ldo=512, lse=0x3000, cu=0x4000, kv_len=0x5000,
             pages=0x6000, ldt=7, max_pages=7, tree=None, S=2, N=9, H=8, scale=0.125):
        return L.kattn_fwd_cached(ctx, cache, dtype, q, ldq, o, ldo, lse, cu, kv_len, pages, ldt, max_pages, tree, S, N, H,
                                  scale, None)

    assert call(ctx=None) == INVALID and call(cache=None) == INVALID
    for kw, status in BAD_CACHES:
        assert call(cache=table(**kw)) == status, kw
    assert call(dtype=4) == UNSUPPORTED
    assert call(H=7) == INVALID and call(H=0) == INVALID
    assert call(S=-1) == INVALID and call(N=-1) == INVALID
    assert call(scale=math.inf) == INVALID
    assert call(ldq=500) == INVALID and call(ldo=516) == MISALIGNED
    assert call(ldt=3) == INVALID and call(ldt=1 << 27, max_pages=1 << 27) == INVALID
    assert call(N=1 << 28) == INVALID
    assert call(tree=0x7004) == MISALIGNED
    for name in ("q", "o", "lse", "cu", "kv_len", "pages"):
        assert call(**{name: None}) == INVALID, name
        assert call(**{name: 0x9002}) == MISALIGNED, name
    assert call(N=0, q=None, o=None, lse=None, cu=None) == 0 and kerr_attn.last_launch_count() == 0


def test_binding_refusals():
    class Fake:
        handle, device = None, 0

    x = torch.zeros(4, 64)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="context on cuda:0"):
        kerr_attn.fwd_packed(Fake, x, x, x, x, torch.zeros(1, 4), i, i, 1)
    with pytest.raises(ValueError):
        kerr_attn.KVCache(torch.zeros(2, 1, 16, 64, dtype=torch.int8), torch.zeros(2, 1, 16, 64, dtype=torch.int8),
                          torch.zeros(2, 1, 16), torch.zeros(2, 1, 16))  # not on a GPU
    with pytest.raises(ValueError):
        kerr_attn.fwd_packed(Fake, x, x, x, x, torch.zeros(1, 4), i, i, 0)
    with pytest.raises(TypeError):
        kerr_attn._dtype_code(torch.zeros(1, dtype=torch.float64), "q")
    for bad, kind in ((lambda: kerr_attn._packed(x.half(), "k", x.dtype, -1, 4, 64), TypeError),
                      (lambda: kerr_attn._packed(x, "k", x.dtype, 0, 4, 64), ValueError),   # another device
                      (lambda: kerr_attn._packed(x, "k", x.dtype, -1, 4, 32), ValueError),  # columns
                      (lambda: kerr_attn._packed(x, "k", x.dtype, -1, 5, 64), ValueError),  # rows
                      (lambda: kerr_attn._packed(x.T, "k", x.dtype, -1, 64, 4), ValueError),
                      (lambda: kerr_attn._ints(i.long(), "cu", 2, -1), ValueError),
                      (lambda: kerr_attn._ints(i, "cu", 3, -1), ValueError),
                      (lambda: kerr_attn._ints(i, "cu", 2, 0), ValueError),
                      (lambda: kerr_attn._sums(torch.zeros(4, 1), 1, 4, -1), ValueError)):
        with pytest.raises(kind):
            bad()
    # A page table whose rows are one row, broadcast.
    class Cache:
        device_index = -1

    row, lengths = torch.zeros(1, 5, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="overlap"):
        kerr_attn._pages(Cache, torch.zeros(4, dtype=torch.int32), lengths, row.expand(3, 5), -1)
    wide = torch.zeros(3, 9, dtype=torch.int32)
    assert kerr_attn._pages(Cache, torch.zeros(4, dtype=torch.int32), lengths, wide[:, :5], -1)[0][3:] == (9, 5)
    assert kerr_attn._pages(Cache, i, lengths[:1], row, -1)[0][3:] == (5, 5)
    assert kerr_attn._packed(x, "k", x.dtype, -1, -1, 64) == 64
    assert kerr_attn._packed(x[:, :32], "k", x.dtype, -1, 4, 32) == 64
    assert kerr_attn._packed(x[:1, :32], "k", x.dtype, -1, 1, 32) == 64


def test_plain_forms_agree():
    # The 64-bit forms: packed rows against one softmax written out; the cache's rounding against a search for the
    # nearest code; attention over a cache against packed rows of what it holds.
    gen = torch.Generator().manual_seed(0)
    H, Hkv, d = 4, 2, 32
    q, k, v = torch.randn(9, H * d, generator=gen), torch.randn(12, Hkv * d, generator=gen), torch.randn(12, Hkv * d, generator=gen)
    o, lse, _, _ = serve_ref.packed(q, k, v, [0, 4, 9], [0, 6, 12], H, Hkv, True, 0.2)
    s = [float(0.2 * (q[5, d:2 * d].double() @ k[6 + j, :d].double())) for j in range(3)]
    w = [math.exp(x) for x in s]
    want = sum(w[j] * v[6 + j, :d].double() for j in range(3)) / sum(w)
    assert (o[5, d:2 * d] - want).abs().max() < 1e-12 and abs(lse[1, 5] - math.log(sum(w))) < 1e-12

    table = torch.cat([torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double() * sign for sign in (1, -1)])
    for fmt, grid in ((0, torch.arange(-127.0, 128).double()), (1, table)):
        x = torch.randn(50, 32, generator=gen) * 5
        codes, scale = serve_ref.quantise(x, fmt)
        inverse = torch.full((50,), serve_ref.LIMIT[fmt]) / x.abs().amax(-1)
        y = x.double() * inverse.double()[:, None]
        assert torch.equal((codes - y).abs(), (grid - y[..., None]).abs().amin(-1))
        assert torch.equal(scale, x.abs().amax(-1) / torch.full((50,), serve_ref.LIMIT[fmt]))

    class Cache:
        page_size, n_pages, n_kv_head, format = 16, 2, Hkv, 0

    Cache.d = d
    codes, scale = serve_ref.quantise(k.view(12, Hkv, d), 0)
    Cache.k = Cache.v = torch.zeros(2, Hkv, 16, d, dtype=torch.int8)
    Cache.k[1, :, :12] = codes.to(torch.int8).transpose(0, 1)
    Cache.k_scale = Cache.v_scale = torch.zeros(2, Hkv, 16)
    Cache.k_scale[1, :, :12] = scale.T
    held = (codes * scale.double()[..., None]).view(12, Hkv * d)
    t = torch.tensor([[1, 0]], dtype=torch.int32)
    a = serve_ref.cached(Cache, q, [0, 9], [12], t, H, None, 0.2)
    b = serve_ref.packed(q, held, held, [0, 9], [0, 12], H, Hkv, True, 0.2)
    assert (a[0] - b[0]).abs().max() < 1e-12 and (a[1] - b[1]).abs().max() < 1e-12
    chain = torch.tensor([(2 << i) - 1 for i in range(9)])
    c = serve_ref.cached(Cache, q, [0, 9], [12], t, H, chain, 0.2)
    assert torch.equal(a[0], c[0])
