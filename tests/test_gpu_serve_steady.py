"""GPU parity of the serving calls in their steady state: every CTA runs through
many items, its rings of tiles, pieces and powers of two come round several
times, and running maxima and units follow ramps.  Against the 64-bit forms,
evaluated on the device; bounds are serve_ref's."""
import math
import random

import pytest
import torch

import kerr_attn
import serve_ref
from test_gpu_serve import TYPES, fill, ints, make_cache, offsets, randn, run_cached, trees

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = kerr_attn.Context(0)
    yield c
    c.check_device()
    c.close()


def check_packed(ctx, q, k, v, nq, nk, H, Hkv, launches, causal=True):
    """fwd_packed in as many launches (1: whole items, 2: parts), against serve_ref.attend sequence by sequence."""
    d = q.shape[1] // H
    cu_q, cu_k = offsets(nq), offsets(nk)
    o = torch.full_like(q, float("nan"))
    lse = torch.full((H, q.shape[0]), float("nan"), device="cuda")
    assert kerr_attn.fwd_packed(ctx, q, k, v, o, lse, ints(cu_q), ints(cu_k), H, Hkv, causal=causal) == launches
    for s, (t, n) in enumerate(zip(nq, nk)):
        a, c = cu_q[s], cu_k[s]
        i, j = torch.arange(t, device="cuda")[:, None], torch.arange(n, device="cuda")
        seen = j <= i + n - t if causal else torch.ones(t, n, dtype=torch.bool, device="cuda")
        want, wl, bo, bl = serve_ref.attend(q[a:a + t].double().view(t, H, d), k[c:c + n].double().view(n, Hkv, d),
                                            v[c:c + n].double().view(n, Hkv, d), seen, 1 / math.sqrt(d), q.dtype)
        serve_ref.check(o[a:a + t].view(t, H, d), want.cpu(), bo.cpu(), f"o of sequence {s}")
        serve_ref.check(lse[:, a:a + t], wl.cpu(), bl.cpu(), f"lse of sequence {s}")


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads", [(8, 8), (9, 3)])
def test_packed_many_whole_items(ctx, heads, dtype, d):
    # Hundreds of items of one to ten steps: more than three for every SM, in sequences of their own magnitudes.
    rng, gen = random.Random(d), torch.Generator().manual_seed(d)
    H, Hkv = heads
    nq = [rng.choice((1, 37, 129, 1000 + rng.randrange(281), rng.randrange(200, 1000))) for _ in range(36)] + [1279, 1, 897]
    nk = list(nq)
    q, k, v = randn(gen, sum(nq), H * d), randn(gen, sum(nk), Hkv * d), randn(gen, sum(nk), Hkv * d)
    cu = offsets(nq)
    for s in range(len(nq)):  # products near one whatever the powers
        up, of_v = 2.0 ** rng.randrange(-9, 10), 2.0 ** rng.randrange(-6, 7)
        q[cu[s]:cu[s + 1]] *= up
        k[cu[s]:cu[s + 1]] /= up
        v[cu[s]:cu[s + 1]] *= of_v
    items = sum(-(-t * (H // Hkv) // 256) for t in nq) * Hkv
    assert items > 3 * 148
    check_packed(ctx, q.to(dtype), k.to(dtype), v.to(dtype), nq, nk, H, Hkv, launches=1)


@pytest.mark.parametrize("way", [1.0, -1.0])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", TYPES)
def test_packed_many_whole_items_over_contexts(ctx, dtype, d, way):
    # Every item walks tens of key tiles while scores and values rise (or fall) along the keys.
    rng, gen = random.Random(d + 1), torch.Generator().manual_seed(d + 1)
    H = Hkv = 6
    nq = [rng.randrange(500, 900) for _ in range(30)]
    nk = [t + rng.randrange(300, 900) for t in nq]
    q, k, v = randn(gen, sum(nq), H * d), randn(gen, sum(nk), Hkv * d), randn(gen, sum(nk), Hkv * d)
    q.view(-1, H, d)[:, :, 0] = 4.0
    ramp = torch.cat([torch.linspace(-way, way, n) for n in nk]).cuda()
    k.view(-1, Hkv, d)[:, :, 0] = 6.0 * ramp[:, None]
    v *= (2.0 ** (6 * ramp))[:, None]
    check_packed(ctx, q.to(dtype), k.to(dtype), v.to(dtype), nq, nk, H, Hkv, launches=1)


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", TYPES)
def test_packed_long_line(ctx, dtype, d):
    # Chunks behind long contexts as one line: parts of several steps, CTAs with the end of one item and the next ones.
    rng, gen = random.Random(d + 2), torch.Generator().manual_seed(d + 2)
    H, Hkv = 6, 3
    nq = [rng.randrange(40, 260) for _ in range(5)] + [1]
    nk = [t + rng.randrange(1500, 5000) for t in nq]
    q, k, v = randn(gen, sum(nq), H * d), randn(gen, sum(nk), Hkv * d), randn(gen, sum(nk), Hkv * d)
    check_packed(ctx, q.to(dtype), k.to(dtype), v.to(dtype), nq, nk, H, Hkv, launches=2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_packed_two_keys(ctx, dtype):
    # Two keys, whose scores differ by up to 2^3: lse is one exponential's, held to its bound at every difference.
    d, n = 64, 4096
    q = torch.zeros(n, d)
    q[:, 0] = torch.arange(n) / 512
    k = torch.zeros(2 * n, d)
    k[::2, 0] = -1.0
    q, k = q.to(dtype).cuda(), k.to(dtype).cuda()
    o, lse = torch.empty_like(q), torch.empty(1, n, device="cuda")
    cu = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    kerr_attn.fwd_packed(ctx, q, k, k, o, lse, cu, 2 * cu, 1, 1, causal=False, scale=1.0)
    x = q[:, 0].double()
    # The products are exact; exp2 is off by 2^-21 and the logarithm, its base and its rounding by 2^-21 and 2^-23 more.
    assert ((lse[0].double() - torch.log1p(torch.exp(-x))).abs() <= 2 * 2.0 ** -21 + 2.0 ** -23).all()


def check_cached(ctx, cache, q, new, kv_len, table, H, tree=None):
    """fwd_cached against serve_ref.attend, sequence by sequence; twice to the same bits."""
    o, lse = run_cached(ctx, cache, q, new, kv_len, table, H, tree)
    again = run_cached(ctx, cache, q, new, kv_len, table, H, tree)
    assert torch.equal(o, again[0]) and torch.equal(lse, again[1])
    cu, d = offsets(new), cache.d
    kind = torch.int8 if cache.format == kerr_attn.CACHE_INT8 else torch.float8_e4m3fn
    for s, (n, length) in enumerate(zip(new, kv_len)):
        if n == 0:
            continue
        j = torch.arange(length, device="cuda")
        page, place = table[s].long()[j // cache.page_size], j % cache.page_size
        k, v = (c.view(kind)[page, :, place].double() * f[page, :, place].double()[..., None]
                for c, f in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
        drafted = j - (length - n)
        a = cu[s]
        if tree is None:
            seen = drafted <= torch.arange(n, device="cuda")[:, None]
        else:
            bits = tree[a:a + n].cuda()[:, None] >> drafted.clamp(0, 63)
            seen = (drafted < 0) | ((bits & 1).bool() & (drafted < 64))
        want, wl, bo, bl = serve_ref.attend(q[a:a + n].double().view(n, H, d), k, v, seen, 1 / math.sqrt(d), q.dtype)
        serve_ref.check(o[a:a + n].view(n, H, d), want.cpu(), bo.cpu(), f"o of sequence {s}")
        serve_ref.check(lse[:, a:a + n], wl.cpu(), bl.cpu(), f"lse of sequence {s}")
    return o, lse


# Query heads, key heads and new tokens: 1, 16 and 60 rows of a key head (row tiles of 8, 16, 32).
ROWS = {"one": (8, 8, 1), "some": (32, 8, 4), "many": (12, 4, 20)}


@pytest.mark.parametrize("way", [0.0, 1.0, -1.0])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", list(ROWS))
def test_cached_long_lines(ctx, name, dtype, d, way):
    # Some ten tiles and more for every CTA; scores and values rise or fall along the positions, or do not.
    H, Hkv, n = ROWS[name]
    if d == 32:
        H, Hkv = 2 * H, 2 * Hkv
    rng, gen = random.Random(d), torch.Generator().manual_seed(d)
    kv_len = [rng.randrange(6000, 10000) for _ in range(7)]
    new = [n, n - 1, n, n, n, n, n]
    fmt = (d // 32 + n) % 2
    page = (16, 64, 256)[n % 3]
    cache, table = make_cache(kv_len, page, Hkv, d, fmt, seed=30)
    cu = offsets(kv_len)
    k, v = randn(gen, cu[-1], Hkv * d), randn(gen, cu[-1], Hkv * d)
    q = randn(gen, sum(new), H * d)
    if way:
        ramp = torch.cat([torch.linspace(-way, way, m) for m in kv_len]).cuda()
        q.view(-1, H, d)[:, :, 0] = 4.0
        k.view(-1, Hkv, d)[:, :, 0] = math.sqrt(d) * ramp[:, None] * 6
        v *= (2.0 ** (6 * ramp))[:, None]
    kerr_attn.cache_append(ctx, cache, k.to(dtype), v.to(dtype), ints(cu), ints(kv_len), table)
    tree = trees(new, 31) if n > 1 else None
    check_cached(ctx, cache, q.to(dtype), new, kv_len, table, H, tree)


@pytest.mark.parametrize("rows", [1, 6, 40])
@pytest.mark.parametrize("dtype", TYPES)
def test_cached_many_pieces(ctx, dtype, rows):
    # Short sequences of many heads: more than five pieces for every CTA.
    rng = random.Random(rows)
    S, H, Hkv, d = 260, 16, 8, 64
    new = [rng.randrange(0, rows + 1) for _ in range(S)]
    kv_len = [t + rng.randrange(0, 200) for t in new]
    cache, table = make_cache(kv_len, 16, Hkv, d, 1, seed=32)
    fill(ctx, cache, table, kv_len, dtype, seed=33)
    q = randn(torch.Generator().manual_seed(34), sum(new), H * d, dtype=dtype)
    pieces = sum(1 for t in new if t) * Hkv
    assert pieces > (5 if rows > 1 else 3) * 296
    check_cached(ctx, cache, q, new, kv_len, table, H, trees(new, 35) if rows == 6 else None)


def test_cache_past_four_gigabytes(ctx):
    # Pages whose codes lie more than 2^32 bytes from the first.
    page, Hkv, d, H = 64, 8, 128, 16
    cache = kerr_attn.KVCache.empty(70000, page, Hkv, d, kerr_attn.CACHE_INT8)
    kv_len, new = [200, 1000], [1, 7]
    pages = list(range(69960, 70000)) + [3, 1]
    random.Random(36).shuffle(pages)
    table = ints([pages[:20], pages[20:40]])
    k, v, cu = fill(ctx, cache, table, kv_len, torch.bfloat16, seed=37)
    q = randn(torch.Generator().manual_seed(38), sum(new), H * d, dtype=torch.bfloat16)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    kerr_attn.cache_read(ctx, cache, ko, vo, ints(cu), ints(kv_len), table)
    for x, out in ((k, ko), (v, vo)):
        codes, scale = serve_ref.quantise(x.view(-1, Hkv, d), 0)
        assert torch.equal(out.cpu(), (codes.float() * scale[..., None]).bfloat16().view(-1, Hkv * d))
    # The same rows on the first pages of a small cache give the same bits.
    small, where = make_cache(kv_len, page, Hkv, d, 0, seed=39)
    kerr_attn.cache_append(ctx, small, k, v, ints(cu), ints(kv_len), where)
    # (a row of the table holds as many entries in both, so that the work is cut alike)
    where = torch.cat([where, torch.full((2, 20 - where.shape[1]), -1, dtype=torch.int32, device="cuda")], 1)
    a = check_cached(ctx, small, q, new, kv_len, where, H)
    b = run_cached(ctx, cache, q, new, kv_len, table, H)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
