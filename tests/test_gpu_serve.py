"""GPU parity of the serving calls (packed prompts, the 8-bit paged cache and
attention over it) with their plain 64-bit forms, at the sizes and masks where
they can go wrong; bounds are serve_ref's."""
import math
import random

import pytest
import torch

import kerr_attn
import serve_ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def ctx():
    c = kerr_attn.Context(0)
    yield c
    c.check_device()
    c.close()


def offsets(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def randn(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen).to(dtype).cuda()


def run_packed(ctx, q, k, v, cu_q, cu_k, H, Hkv, causal=True, scale=None, stream=None):
    o = torch.full_like(q, float("nan"))
    lse = torch.full((H, q.shape[0]), float("nan"), device="cuda")
    kerr_attn.fwd_packed(ctx, q, k, v, o, lse, ints(cu_q), ints(cu_k), H, Hkv, causal=causal, scale=scale, stream=stream)
    return o, lse


def check_packed(ctx, q, k, v, cu_q, cu_k, H, Hkv, causal=True, scale=None):
    d = q.shape[1] // H
    sc = 1 / math.sqrt(d) if scale is None else scale
    o, lse = run_packed(ctx, q, k, v, cu_q, cu_k, H, Hkv, causal, scale)
    want, wl, bo, bl = serve_ref.packed(q, k, v, cu_q, cu_k, H, Hkv, causal, sc)
    serve_ref.check(o, want, bo, "o")
    serve_ref.check(lse, wl, bl, "lse")
    # Rows of keys behind the last sequence's make the work look long: it is cut into parts.
    o2, lse2 = run_packed(ctx, q, *(long_rows(x, len(cu_q) - 1) for x in (k, v)), cu_q, cu_k, H, Hkv, causal, scale)
    serve_ref.check(o2, want, bo, "o in parts")
    serve_ref.check(lse2, wl, bl, "lse in parts")
    return o, lse


def long_rows(x, sequences):
    return torch.cat([x, torch.full((4000 * sequences, x.shape[1]), float("nan"), dtype=x.dtype, device="cuda")])


# Query rows, key rows (None: the same), query and key heads of each sequence.
PACKED = {
    "one": ([1], None, 1, 1),
    "ragged": ([5, 0, 130, 1, 64], None, 4, 4),
    "group3": ([129, 257, 63], None, 6, 2),
    "group5": ([1, 200, 40], None, 5, 1),
    "group8": ([300, 7, 128], None, 8, 1),
    "chunks": ([3, 128, 17, 1], [300, 129, 17, 513], 4, 2),
    "fewer_keys": ([40, 200, 9], [10, 0, 9], 2, 1),
    "longer": ([700, 1030], None, 2, 1),
    "far_context": ([3, 200, 0, 40], [2000, 3500, 300, 2600], 4, 2),
}


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", list(PACKED))
def test_packed(ctx, name, dtype, d):
    nq, nk, H, Hkv = PACKED[name]
    nk = nq if nk is None else nk
    gen = torch.Generator().manual_seed(1)
    q = randn(gen, sum(nq), H * d, dtype=dtype)
    k, v = (randn(gen, sum(nk), Hkv * d, dtype=dtype) for _ in range(2))
    check_packed(ctx, q, k, v, offsets(nq), offsets(nk), H, Hkv)


@pytest.mark.parametrize("dtype", TYPES)
def test_packed_every_key(ctx, dtype):
    gen = torch.Generator().manual_seed(2)
    nq, nk, H, Hkv, d = [70, 1, 300], [200, 129, 5], 4, 2, 64
    q = randn(gen, sum(nq), H * d, dtype=dtype)
    k, v = (randn(gen, sum(nk), Hkv * d, dtype=dtype) for _ in range(2))
    check_packed(ctx, q, k, v, offsets(nq), offsets(nk), H, Hkv, causal=False, scale=0.3)


@pytest.mark.parametrize("order", ["rising", "falling", "far"])
@pytest.mark.parametrize("dtype", TYPES)
def test_packed_running_maximum(ctx, dtype, order):
    # Scores whose row maximum keeps rising from tile to tile, falls, or lies hundreds away.
    gen = torch.Generator().manual_seed(3)
    n, H, d = 600, 1, 64
    q = torch.ones(n, d) * 0.5
    ramp = torch.linspace(-1, 1, n)[:, None] * (20.0 if order == "far" else 4.0)
    k = (ramp if order != "falling" else -ramp) + 0.05 * torch.randn(n, d, generator=gen)
    v = torch.randn(n, d, generator=gen)
    q, k, v = (x.to(dtype).cuda() for x in (q, k, v))
    check_packed(ctx, q, k, v, [0, n], [0, n], H, H, scale=1.0)
    check_packed(ctx, q, k, v, [0, n], [0, n], H, H, scale=-1.0)
    check_packed(ctx, q, k, v, [0, n], [0, n], H, H, scale=0.0)


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("v_from,v_to", [(-30, 30), (30, -30), (0, 12), (-38, -38), (37, 37)])
def test_packed_f32_magnitudes(ctx, v_from, v_to, d):
    # Far powers of ten: v's from the first key to the last, q's and k's by row (their products near one),
    # one column of each a thousand times the others.
    gen = torch.Generator().manual_seed(8)
    n, H = 500, 2
    q, k, v = (torch.randn(n, H * d, generator=gen) for _ in range(3))
    v = v.clamp(-3, 3) * torch.logspace(v_from, v_to, n, dtype=torch.float64)[:, None].float()
    q[:, 3] *= 1e3
    k[:, 5] *= 1e3
    v[:, 7] *= 1e3 if v_to < 30 and v_from < 30 else 1e-3
    up = 10.0 ** (16 * torch.rand(1, generator=gen).item())
    check_packed(ctx, (q * up).cuda(), (k / up).cuda(), v.cuda(), [0, 200, n], [0, 200, n], H, H)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [32, 128])
def test_packed_strides_and_padding(ctx, dtype, d):
    # q, k and v are column blocks of one buffer, o a block of a wider one; the arrays hold rows before the first and
    # behind the last sequence, full of NaN on the way in and left as they were on the way out.
    gen = torch.Generator().manual_seed(4)
    H, Hkv, nq = 4, 2, [33, 140]
    cu, N = [6, 39, 179], 200
    buf = randn(gen, N, (H + 2 * Hkv) * d + 16, dtype=dtype)
    buf[:6] = float("nan")
    buf[179:] = float("nan")
    q, k, v = buf[:, :H * d], buf[:, H * d:(H + Hkv) * d], buf[:, (H + Hkv) * d:(H + 2 * Hkv) * d]
    wide = torch.full((N, 2 * H * d), 7.0, dtype=dtype, device="cuda")
    lse = torch.full((H, N), 7.0, device="cuda")
    kerr_attn.fwd_packed(ctx, q, k, v, wide[:, :H * d], lse, ints(cu), ints(cu), H, Hkv)
    want, wl, bo, bl = serve_ref.packed(q, k, v, cu, cu, H, Hkv, True, 1 / math.sqrt(d))
    serve_ref.check(wide[:, :H * d], want, bo, "o")
    serve_ref.check(lse, wl, bl, "lse")
    assert (wide[:, H * d:] == 7).all() and (wide[:6] == 7).all() and (wide[179:] == 7).all()
    assert (lse[:, :6] == 7).all() and (lse[:, 179:] == 7).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype", TYPES)
def test_packed_bad_values_stay_in_their_sequence(ctx, dtype, bad):
    gen = torch.Generator().manual_seed(5)
    H, Hkv, d, nq = 2, 1, 64, [50, 21, 200, 3, 90]
    cu = offsets(nq)
    q = randn(gen, sum(nq), H * d, dtype=dtype)
    k, v = (randn(gen, sum(nq), Hkv * d, dtype=dtype) for _ in range(2))
    clean, cl = run_packed(ctx, q, k, v, cu, cu, H, Hkv)
    for s in (1, 3):
        for x in (q, k, v):
            x[cu[s]:cu[s + 1]] = bad
    o, lse = run_packed(ctx, q, k, v, cu, cu, H, Hkv)
    for s in (0, 2, 4):
        assert torch.equal(o[cu[s]:cu[s + 1]], clean[cu[s]:cu[s + 1]])
        assert torch.equal(lse[:, cu[s]:cu[s + 1]], cl[:, cu[s]:cu[s + 1]])


def test_packed_broken_offsets_stay_inside(ctx):
    # Offsets that descend or leave the arrays are brought inside: no row outside is touched.
    H, d, N = 2, 64, 100
    q = torch.randn(N, H * d, device="cuda")
    guard = torch.full((N + 40, H * d), 3.0, device="cuda")
    o, lse = guard[20:20 + N], torch.zeros(H, N, device="cuda")
    kerr_attn.fwd_packed(ctx, q, q, q, o, lse, ints([0, 500, 40, -7, 1000]), ints([-90, 60, 20, 400, 100]), H, H)
    torch.cuda.synchronize()
    assert (guard[:20] == 3).all() and (guard[20 + N:] == 3).all()


@pytest.mark.parametrize("sequences,keys", [(200, 1000), (200, 400000), (3000, 1000)])
def test_packed_overlapping_offsets_stay_inside(ctx, sequences, keys):
    # Offsets that rise and fall: every other sequence owns all rows, far more items than rows make.
    H, Hkv, d, N = 4, 1, 64, 1000
    q, k = torch.randn(N, H * d, device="cuda"), torch.randn(keys, Hkv * d, device="cuda")
    guard = torch.full((N + 40, H * d), 3.0, device="cuda")
    o, lse = guard[20:20 + N], torch.zeros(H, N, device="cuda")
    cu = ints([0, N] * sequences)
    kerr_attn.fwd_packed(ctx, q, k, k, o, lse, cu, cu, H, Hkv)
    torch.cuda.synchronize()
    assert (guard[:20] == 3).all() and (guard[20 + N:] == 3).all()


def test_packed_wide_group_long(ctx):
    # Rows times the group's heads past 2^32 / group: every row sees the one key.
    gen = torch.Generator(device="cuda").manual_seed(9)
    H, d, n = 512, 32, 18000
    q = torch.randn(n, H * d, device="cuda", generator=gen).bfloat16()
    k, v = (torch.randn(1, d, device="cuda", generator=gen).bfloat16() for _ in range(2))
    o, lse = torch.full_like(q, 7.0), torch.zeros(H, n, device="cuda")
    kerr_attn.fwd_packed(ctx, q, k, v, o, lse, ints([0, n]), ints([0, 1]), H, 1, causal=False, scale=1.0)
    assert torch.equal(o.view(n, H, d), v.expand(n, H, d))
    exact = q.view(n, H, d).double() @ k[0].double()
    most = q.view(n, H, d).double().abs() @ k[0].double().abs()
    assert ((lse.T - exact).abs() <= (d + 3) * 2.0 ** -24 * most + 2.0 ** -20 + 2.0 ** -22 * exact.abs()).all()


def test_packed_far_rows(ctx):
    # Rows further apart than 2^31 elements.
    gen = torch.Generator().manual_seed(6)
    N, H, d, ld = 70, 1, 32, 1 << 25
    big = torch.zeros(N * ld, dtype=torch.bfloat16, device="cuda").view(N, ld)
    q, k, v, o = (big[:, i * d:(i + 1) * d] for i in range(4))
    for x in (q, k, v):
        x.copy_(randn(gen, N, d, dtype=torch.bfloat16))
    lse = torch.empty(H, N, device="cuda")
    kerr_attn.fwd_packed(ctx, q, k, v, o, lse, ints([0, 3, N]), ints([0, 3, N]), H, H)
    want, wl, bo, bl = serve_ref.packed(q, k, v, [0, 3, N], [0, 3, N], H, H, True, 1 / math.sqrt(d))
    serve_ref.check(o, want, bo, "o")
    serve_ref.check(lse, wl, bl, "lse")


def test_packed_matches_the_square_batch(ctx):
    # One batch of equal lengths through kattn_fwd and as packed rows.
    gen = torch.Generator().manual_seed(7)
    B, T, H, d = 3, 130, 4, 64
    qkv = randn(gen, B, T, 3 * H * d)
    q, k, v = kerr_attn.split_qkv(qkv, H * d)
    o, lse = torch.empty(B, T, H * d, device="cuda"), torch.empty(B, H, T, device="cuda")
    kerr_attn.fwd(ctx, q, k, v, o, lse, H)
    cu = [0, T, 2 * T, 3 * T]
    flat = qkv.view(B * T, -1)
    po, pl = run_packed(ctx, *(x.squeeze(0) for x in (flat[None, :, :H * d], flat[None, :, H * d:2 * H * d],
                                                      flat[None, :, 2 * H * d:])), cu, cu, H, H)
    # Both are within 1e-4 of the formula (the bar of the parity tests).
    assert (po.view(B, T, -1) - o).abs().max() < 2e-4 * o.abs().max()
    assert (pl.view(H, B, T).transpose(0, 1) - lse).abs().max() < 2e-4


# ------------------------------------------------------------------ the cache

def make_cache(kv_len, page, Hkv, d, fmt, seed, spare=2):
    """A cache and a shuffled page table; a sequence's unused entries lie outside the cache."""
    used = [-(-max(n, 0) // page) for n in kv_len]
    total = sum(used) + spare
    order = list(range(total))
    random.Random(seed).shuffle(order)
    table, at = [], 0
    width = max(used + [1]) + 1
    for u in used:
        table.append(order[at:at + u] + [-1 if at % 2 else total] * (width - u))
        at += u
    return kerr_attn.KVCache.empty(total, page, Hkv, d, fmt), ints(table)


def fill(ctx, cache, table, kv_len, dtype, seed):
    """Whole sequences of random rows appended; keys with a few large channels."""
    gen = torch.Generator().manual_seed(seed)
    cu = offsets([max(n, 0) for n in kv_len])
    cols = cache.n_kv_head * cache.d
    wide = 1 + 3 * (torch.rand(cols, generator=gen) < 0.05)
    k, v = (torch.randn(cu[-1], cols, generator=gen) * wide).to(dtype).cuda(), randn(gen, cu[-1], cols, dtype=dtype)
    kerr_attn.cache_append(ctx, cache, k, v, ints(cu), ints(kv_len), table)
    return k, v, cu


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("fmt", [kerr_attn.CACHE_INT8, kerr_attn.CACHE_E4M3])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", TYPES)
def test_cache_append_and_read(ctx, dtype, d, fmt, page):
    kv_len, Hkv = [1, 37, 16, 0, 300, 257], 3
    cache, table = make_cache(kv_len, page, Hkv, d, fmt, seed=d + page)
    before = [x.clone() for x in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    k, v, cu = fill(ctx, cache, table, kv_len, dtype, seed=8)
    got = serve_ref.values(cache)
    want, scales = [torch.zeros_like(x) for x in got], [x.cpu().clone() for x in before[2:]]
    for x, c, s in ((k, want[0], scales[0]), (v, want[1], scales[1])):
        codes, scale = serve_ref.quantise(x.view(-1, Hkv, d), fmt)
        for i, n in enumerate(kv_len):
            for p in range(n):
                page_, place = serve_ref.position(cache, table.cpu(), i, p)
                c[page_, :, place] = codes[cu[i] + p]
                s[page_, :, place] = scale[cu[i] + p]
    # Codes and scales are exact; every other place keeps what it held.
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(cache.k_scale.cpu(), scales[0]) and torch.equal(cache.v_scale.cpu(), scales[1])
    # Read whole sequences, and the last few positions of each.
    for take in (kv_len, [min(n, 5) for n in kv_len]):
        cr = offsets(take)
        ko, vo = (torch.full((cr[-1] + 3, Hkv * d), 9.0, dtype=dtype, device="cuda") for _ in range(2))
        kerr_attn.cache_read(ctx, cache, ko, vo, ints(cr), ints(kv_len), table)
        for x, out in ((k, ko), (v, vo)):
            codes, scale = serve_ref.quantise(x.view(-1, Hkv, d), fmt)
            held = (codes.float() * scale[..., None]).to(dtype).view(-1, Hkv * d)
            rows = torch.cat([torch.arange(cu[i + 1] - t, cu[i + 1]) for i, t in enumerate(take)])
            assert torch.equal(out[:cr[-1]].cpu(), held[rows])
            assert (out[cr[-1]:] == 9).all()


@pytest.mark.parametrize("fmt", [kerr_attn.CACHE_INT8, kerr_attn.CACHE_E4M3])
@pytest.mark.parametrize("dtype", TYPES)
def test_cache_borders_of_the_codes(ctx, dtype, fmt):
    # Values in the middle between two codes, just beside it, and rows of nothing, of tiny, huge and bad numbers.
    d, page = 32, 16
    limit = serve_ref.LIMIT[fmt]
    rows = []
    if fmt == kerr_attn.CACHE_INT8:
        middles = torch.arange(-126.5, 127, 1.0)
    else:
        table = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
        middles = ((table[1:] + table[:-1]) / 2).float()
    for i in range(0, len(middles), 31):
        part = middles[i:i + 31]
        for nudge in (0.0, 1e-7, -1e-7, 2e-3, -2e-3):
            x = torch.zeros(d)
            x[0] = limit
            x[1:1 + len(part)] = part * (1 + nudge)
            rows += [x, x * 0.37, -x * 2.0 ** -7]
    rows += [torch.zeros(d), torch.full((d,), 1e-38), torch.full((d,), 6e4), torch.linspace(-3, 3, d)]
    for bad in (float("nan"), float("inf"), -float("inf")):
        x = torch.linspace(-1, 1, d)
        x[7] = bad
        rows.append(x)
    k = torch.stack(rows).to(dtype).cuda()
    n = k.shape[0]
    cache, table = make_cache([n], page, 1, d, fmt, seed=1)
    kerr_attn.cache_append(ctx, cache, k, -k, ints([0, n]), ints([n]), table)
    ko, vo = torch.empty_like(k), torch.empty_like(k)
    kerr_attn.cache_read(ctx, cache, ko, vo, ints([0, n]), ints([n]), table)
    codes, scale = serve_ref.quantise(k, fmt)
    held = (codes.float() * scale[..., None]).to(dtype)
    assert torch.equal(ko.cpu().nan_to_num(777.0), held.nan_to_num(777.0))
    assert torch.equal(vo.cpu().nan_to_num(777.0), (-held).nan_to_num(777.0))
    assert torch.isnan(ko[-3:]).all() and not torch.isnan(ko[:-3]).any()


def test_cache_places_that_do_not_exist(ctx):
    # Bad pages, positions before zero and past the table: nothing is written, zeros are read.
    page, Hkv, d = 16, 2, 64
    cache = kerr_attn.KVCache.empty(3, page, Hkv, d)
    table = ints([[1, 3], [-1, 0], [2, 2]])
    kv_len, cu = ints([32, 32, 50]), [0, 32, 64, 114]
    k = torch.randn(120, Hkv * d, device="cuda")
    kerr_attn.cache_append(ctx, cache, k, k, ints(cu), kv_len, table)
    ko, vo = (torch.full_like(k, 9.0) for _ in range(2))
    kerr_attn.cache_read(ctx, cache, ko, vo, ints(cu), kv_len, table)
    codes, scale = serve_ref.quantise(k.view(-1, Hkv, d), 0)
    held = (codes.float() * scale[..., None]).view(-1, Hkv * d)
    ko = ko.cpu()
    assert torch.equal(ko[:16], held[:16]) and (ko[16:32] == 0).all()       # page 3 of 3
    assert (ko[32:48] == 0).all() and torch.equal(ko[48:64], held[48:64])   # page -1
    assert (ko[96:114] == 0).all() and (ko[114:] == 9).all()                # positions past two pages; no sequence's rows
    # A length below its rows: the first rows lie before position zero.
    cache.k.zero_()
    kerr_attn.cache_append(ctx, cache, k[:20], k[:20], ints([0, 20]), ints([12]), table[:1])
    kerr_attn.cache_read(ctx, cache, vo[:20], vo[20:40], ints([0, 20]), ints([12]), table[:1])
    assert (vo[:8] == 0).all() and torch.equal(vo[8:20].cpu(), held[8:20])


# ------------------------------------------------------------------ attention over the cache

def trees(lengths, seed, empty=False):
    """Random trees as bits; with `empty`, some rows that see no drafted token."""
    rng, words = random.Random(seed), []
    for n in lengths:
        mine = []
        for j in range(n):
            parent = rng.randrange(-1, j) if j else -1
            word = (mine[parent] if 0 <= parent < 64 else 0) | (1 << j if j < 64 else 0)
            mine.append(word)
        words += [0 if empty and i % 3 == 1 else w for i, w in enumerate(mine)]
    return torch.tensor([w - (1 << 64) if w >> 63 else w for w in words], dtype=torch.int64)


def run_cached(ctx, cache, q, new, kv_len, table, H, tree=None, scale=None):
    cu = offsets(new)
    o = torch.full_like(q, float("nan"))
    lse = torch.full((H, q.shape[0]), float("nan"), device="cuda")
    kerr_attn.fwd_cached(ctx, cache, q, o, lse, ints(cu), ints(kv_len), table, H,
                         tree=None if tree is None else tree.cuda(), scale=scale)
    return o, lse


def check_cached(ctx, cache, q, new, kv_len, table, H, tree=None, scale=None):
    o, lse = run_cached(ctx, cache, q, new, kv_len, table, H, tree, scale)
    sc = 1 / math.sqrt(cache.d) if scale is None else scale
    want, wl, bo, bl = serve_ref.cached(cache, q, offsets(new), kv_len, table, H, tree, sc)
    serve_ref.check(o, want, bo, "o")
    serve_ref.check(lse, wl, bl, "lse")
    return o, lse


# New tokens and lengths of each sequence, query and key heads, page size, whether a tree.
CACHED = {
    "first_token": ([1], [1], 1, 1, 16, False),
    "decode": ([1, 1, 1, 1], [1, 16, 17, 700], 12, 12, 16, False),
    "group4": ([1, 0, 1], [333, 40, 129], 8, 2, 64, False),
    "group5": ([1, 1], [64, 1000], 5, 1, 256, False),
    "chain": ([3, 1, 8, 20], [3, 90, 300, 65], 4, 2, 32, False),
    "long_chain": ([150], [400], 3, 1, 16, False),
    "trees": ([5, 64, 1, 33], [200, 64, 31, 600], 4, 1, 16, True),
    "group8_trees": ([16, 7], [900, 129], 16, 2, 128, True),
    "past_64": ([70], [130], 2, 2, 16, True),
}


@pytest.mark.parametrize("fmt", [kerr_attn.CACHE_INT8, kerr_attn.CACHE_E4M3])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", list(CACHED))
def test_cached(ctx, name, dtype, d, fmt):
    new, kv_len, H, Hkv, page, tree = CACHED[name]
    cache, table = make_cache(kv_len, page, Hkv, d, fmt, seed=3)
    fill(ctx, cache, table, kv_len, dtype, seed=9)
    q = randn(torch.Generator().manual_seed(10), sum(new), H * d, dtype=dtype)
    check_cached(ctx, cache, q, new, kv_len, table, H, trees(new, 4) if tree else None)


@pytest.mark.parametrize("dtype", TYPES)
def test_cached_rows_that_see_nothing(ctx, dtype):
    # Empty tree rows of sequences without earlier tokens, lengths of zero, pages that do not exist.
    new, kv_len, H, Hkv, d = [6, 4, 3, 2], [6, 0, 40, 30], 4, 2, 64
    cache, table = make_cache(kv_len, 16, Hkv, d, 0, seed=5)
    fill(ctx, cache, table, kv_len, dtype, seed=11)
    table[3] = -5
    q = randn(torch.Generator().manual_seed(12), sum(new), H * d, dtype=dtype)
    o, lse = check_cached(ctx, cache, q, new, kv_len, table, H, trees(new, 6, empty=True))
    assert (o[6:10] == 0).all() and (lse[:, 6:10] == -math.inf).all()
    assert (o[13:] == 0).all() and (lse[:, 13:] == -math.inf).all()
    assert (o[1] == 0).all() and (lse[:, 1] == -math.inf).all()


@pytest.mark.parametrize("fmt", [kerr_attn.CACHE_INT8, kerr_attn.CACHE_E4M3])
@pytest.mark.parametrize("dtype", TYPES)
def test_cached_large_and_small_numbers(ctx, dtype, fmt):
    # Queries, keys and values far from one, values whose scales differ by a million within a sequence.
    gen = torch.Generator().manual_seed(13)
    new, kv_len, H, Hkv, d = [2, 1], [500, 77], 2, 1, 64
    cache, table = make_cache(kv_len, 16, Hkv, d, fmt, seed=6)
    cu = offsets(kv_len)
    k = torch.randn(cu[-1], d, generator=gen) * 30
    v = torch.randn(cu[-1], d, generator=gen) * torch.where(torch.arange(cu[-1]) % 3 == 0, 1e3, 1e-3)[:, None]
    k, v = k.to(dtype).cuda(), v.to(dtype).cuda()
    kerr_attn.cache_append(ctx, cache, k, v, ints(cu), ints(kv_len), table)
    for size, scale in ((1.0, 0.1), (1e-3, 1.0), (200.0, 1e-3), (1.0, -0.1), (1.0, 0.0)):
        q = (torch.randn(3, H * d, generator=gen) * size).to(dtype).cuda()
        check_cached(ctx, cache, q, new, kv_len, table, H, scale=scale)


@pytest.mark.parametrize("dtype", TYPES)
def test_cached_bad_values_in_unseen_places(ctx, dtype):
    # Poisoned rows (a NaN or an infinity when they were written) reach only the rows that see them.
    new, kv_len, H, Hkv, d = [4, 1], [40, 90], 4, 2, 64
    cache, table = make_cache(kv_len, 16, Hkv, d, 0, seed=7)
    k, v, cu = fill(ctx, cache, table, kv_len, dtype, seed=14)
    tree = torch.tensor([1, 3, 5, 9, 1], dtype=torch.int64)
    q = randn(torch.Generator().manual_seed(15), 5, H * d, dtype=dtype)
    clean, cl = run_cached(ctx, cache, q, new, kv_len, table, H, tree)
    k[cu[0] + 37, 3] = float("nan")  # drafted token 1, seen by row 1 alone
    v[cu[0] + 38, 5] = float("inf")  # drafted token 2, seen by row 2 alone
    kerr_attn.cache_append(ctx, cache, k, v, ints(cu), ints(kv_len), table)
    o, lse = run_cached(ctx, cache, q, new, kv_len, table, H, tree)
    for r in (0, 3, 4):
        assert torch.equal(o[r], clean[r]) and torch.equal(lse[:, r], cl[:, r])
    assert torch.isnan(o[1, :2 * d]).all() and torch.isnan(lse[:2, 1]).all()
    assert torch.isnan(o[2, :2 * d]).all()
    # What lies in places that no position of the batch has does not matter.
    held = {int(p) for row, n in zip(table.cpu(), kv_len) for p in row[:-(-n // 16)]}
    for p in range(cache.n_pages):
        if p not in held:
            cache.k_scale[p] = float("nan")
            cache.v_scale[p] = float("inf")
    last = int(table[1, 90 // 16])
    cache.k_scale[last, :, 90 % 16:] = float("nan")
    cache.v_scale[last, :, 90 % 16:] = float("nan")
    again, al = run_cached(ctx, cache, q, new, kv_len, table, H, tree)
    assert torch.equal(again[4], clean[4]) and torch.equal(al[:, 4], cl[:, 4])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_cached_long_and_ragged(ctx, dtype):
    # A long sequence beside short ones: its parts are joined, twice to the same bits.
    new, kv_len, H, Hkv, d = [1, 3, 1, 2], [5000, 3, 70, 900], 8, 2, 128
    cache, table = make_cache(kv_len, 32, Hkv, d, 1, seed=8)
    fill(ctx, cache, table, kv_len, dtype, seed=16)
    q = randn(torch.Generator().manual_seed(17), sum(new), H * d, dtype=dtype)
    o, lse = check_cached(ctx, cache, q, new, kv_len, table, H)
    o2, lse2 = run_cached(ctx, cache, q, new, kv_len, table, H)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)


def test_cached_many_sequences(ctx):
    rng = random.Random(18)
    S, H, Hkv, d = 300, 4, 2, 32
    new = [rng.choice((0, 1, 1, 1, 2)) for _ in range(S)]
    kv_len = [n + rng.randrange(0, 80) for n in new]
    cache, table = make_cache(kv_len, 16, Hkv, d, 0, seed=9)
    fill(ctx, cache, table, kv_len, torch.bfloat16, seed=19)
    q = randn(torch.Generator().manual_seed(20), sum(new), H * d, dtype=torch.bfloat16)
    check_cached(ctx, cache, q, new, kv_len, table, H)


def test_cached_strides_and_padding(ctx):
    # q and o are blocks of wider buffers, the table a part of a wider one; rows of no sequence stay.
    H, Hkv, d, N = 4, 2, 64, 9
    kv_len, cu = [50, 20], [2, 5, 7]
    cache, table = make_cache(kv_len, 16, Hkv, d, 0, seed=10)
    fill(ctx, cache, table, kv_len, torch.float32, seed=21)
    wide = torch.full((2, 40), -9, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    buf = torch.randn(N, 3 * H * d, device="cuda")
    buf[:2] = float("nan")
    buf[7:] = float("nan")
    out = torch.full((N, 2 * H * d), 7.0, device="cuda")
    lse = torch.full((H, N), 7.0, device="cuda")
    kerr_attn.fwd_cached(ctx, cache, buf[:, H * d:2 * H * d], out[:, H * d:], lse, ints(cu), ints(kv_len), wide[:, :7], H)
    want, wl, bo, bl = serve_ref.cached(cache, buf[:, H * d:2 * H * d], cu, kv_len, wide[:, :7], H, None, 1 / math.sqrt(d))
    serve_ref.check(out[:, H * d:], want, bo, "o")
    serve_ref.check(lse, wl, bl, "lse")
    assert (out[:, :H * d] == 7).all() and (out[:2] == 7).all() and (out[7:] == 7).all()
    assert (lse[:, :2] == 7).all() and (lse[:, 7:] == 7).all()


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("fmt", [kerr_attn.CACHE_INT8, kerr_attn.CACHE_E4M3])
def test_prompt_then_steps_then_a_tree(ctx, dtype, fmt):
    """Prompts in two chunks (the second over the cache read back), two decoded
    tokens and a tree of drafted ones, each against attention over what the cache holds."""
    gen = torch.Generator().manual_seed(22)
    H, Hkv, d, page = 6, 2, 64, 32
    prompts = [[100, 37], [20, 1], [7, 130]]  # two chunks of each
    steps = [[1, 1, 1], [1, 1, 1], [9, 5, 12]]
    final = [sum(p) + 2 + t for p, t in zip(prompts, steps[2])]
    cache, table = make_cache(final, page, Hkv, d, fmt, seed=11)
    kv_len = [0, 0, 0]
    scale = 1 / math.sqrt(d)
    for chunk in range(2):
        new = [p[chunk] for p in prompts]
        kv_len = [a + b for a, b in zip(kv_len, new)]
        cu, cu_k = offsets(new), offsets(kv_len)
        q = randn(gen, sum(new), H * d, dtype=dtype)
        k, v = (randn(gen, sum(new), Hkv * d, dtype=dtype) for _ in range(2))
        kerr_attn.cache_append(ctx, cache, k, v, ints(cu), ints(kv_len), table)
        ka, va = (torch.empty(sum(kv_len), Hkv * d, dtype=dtype, device="cuda") for _ in range(2))
        kerr_attn.cache_read(ctx, cache, ka, va, ints(cu_k), ints(kv_len), table)
        o, lse = check_packed(ctx, q, ka, va, cu, cu_k, H, Hkv)
        # The same rows over the cache itself; bounds of both, and of the values' rounding to the type (u each).
        want, wl, bo, bl = serve_ref.cached(cache, q, cu, kv_len, table, H, None, scale)
        got, gl = run_cached(ctx, cache, q, new, kv_len, table, H)
        serve_ref.check(got, want, bo, "o over the cache")
        serve_ref.check(gl, wl, bl, "lse over the cache")
    for i, new in enumerate(steps):
        kv_len = [a + b for a, b in zip(kv_len, new)]
        q = randn(gen, sum(new), H * d, dtype=dtype)
        k, v = (randn(gen, sum(new), Hkv * d, dtype=dtype) for _ in range(2))
        kerr_attn.cache_append(ctx, cache, k, v, ints(offsets(new)), ints(kv_len), table)
        check_cached(ctx, cache, q, new, kv_len, table, H, trees(new, 7) if i == 2 else None)
    assert kv_len == final


def test_captured_steps_follow_their_lengths(ctx):
    """Two captured decoding steps of the same buffers, replayed with lengths,
    tables and rows that changed, on another stream than the inputs were made
    on, one graph running behind the other."""
    H, Hkv, d, page, S, N = 4, 2, 64, 16, 3, 12
    cache, table = make_cache([400, 400, 400], page, Hkv, d, 0, seed=12)
    gen = torch.Generator().manual_seed(23)
    q = randn(gen, N, H * d)
    long_k, long_v = (long_rows(randn(gen, N, Hkv * d), S) for _ in range(2))  # packed work in parts: a workspace
    k, v = long_k[:N], long_v[:N]
    cu, kv_len = ints([0, 1, 2, 3]), ints([1, 1, 1])
    outs = [(torch.zeros_like(q), torch.zeros(H, N, device="cuda")) for _ in range(2)]
    packed = (torch.zeros_like(q), torch.zeros(H, N, device="cuda"))
    side = torch.cuda.Stream()
    graphs = []
    torch.cuda.synchronize()
    for o, lse in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            kerr_attn.cache_append(ctx, cache, k, v, cu, kv_len, table)
            kerr_attn.fwd_cached(ctx, cache, q, o, lse, cu, kv_len, table, H)
            kerr_attn.fwd_packed(ctx, q, long_k, long_v, *packed, cu, cu, H, Hkv)
        graphs.append(g)
    length = [0, 0, 0]
    for turn, new in enumerate(([4, 2, 3], [1, 1, 1], [5, 0, 7], [2, 2, 2], [1, 1, 1])):
        length = [a + b for a, b in zip(length, new)]
        with torch.cuda.stream(side):
            for x in (q, k, v):
                x.copy_(randn(gen, *x.shape))
            cu.copy_(ints(offsets(new)))
            kv_len.copy_(ints(length))
            for o, lse in outs:
                o.fill_(5)
            graphs[turn % 2].replay()
            graphs[1 - turn % 2].replay()
        side.synchronize()
        want, wl, bo, bl = serve_ref.cached(cache, q, offsets(new), length, table, H, None, 1 / math.sqrt(d))
        for o, lse in outs:
            serve_ref.check(o, want, bo, "o")
            serve_ref.check(lse, wl, bl, "lse")
            assert (o[sum(new):] == 5).all()
        want, wl, bo, bl = serve_ref.packed(q, k, v, offsets(new), offsets(new), H, Hkv, True, 1 / math.sqrt(d))
        serve_ref.check(packed[0], want, bo, "packed o")
    del graphs


def test_two_streams_at_once(ctx):
    # Calls of one context on two streams share no workspace.
    H, Hkv, d, page = 8, 2, 128, 64
    jobs = []
    for i in range(2):
        kv_len = [3000 + 500 * i, 40]
        cache, table = make_cache(kv_len, page, Hkv, d, i, seed=13 + i)
        fill(ctx, cache, table, kv_len, torch.bfloat16, seed=24 + i)
        q = randn(torch.Generator().manual_seed(26 + i), 4, H * d, dtype=torch.bfloat16)
        k = randn(torch.Generator().manual_seed(28 + i), 3000, Hkv * d)
        jobs.append((cache, table, kv_len, q, k, run_cached(ctx, cache, q, [3, 1], kv_len, table, H),
                     run_packed(ctx, torch.cat([k[:500]] * 4, 1), k, k, [0, 500], [0, 3000], H, Hkv)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            cache, table, kv_len, q, k, _, _ = jobs[i]
            with torch.cuda.stream(s):
                got[i].append((run_cached(ctx, cache, q, [3, 1], kv_len, table, H),
                               run_packed(ctx, torch.cat([k[:500]] * 4, 1), k, k, [0, 500], [0, 3000], H, Hkv)))
    torch.cuda.synchronize()
    for i in range(2):
        for a, b in got[i]:
            assert torch.equal(a[0], jobs[i][5][0]) and torch.equal(a[1], jobs[i][5][1])
            assert torch.equal(b[0], jobs[i][6][0]) and torch.equal(b[1], jobs[i][6][1])


def test_nothing_to_do(ctx):
    q, lse = torch.empty(0, 64, device="cuda"), torch.empty(1, 0, device="cuda")
    assert kerr_attn.fwd_packed(ctx, q, q, q, q, lse, ints([0]), ints([0]), 1) == 0
    cache = kerr_attn.KVCache.empty(2, 16, 1, 64)
    none = torch.empty(0, 3, dtype=torch.int32, device="cuda")
    assert kerr_attn.cache_append(ctx, cache, q, q, ints([0]), ints([]), none) == 0
    assert kerr_attn.cache_read(ctx, cache, q, q, ints([0]), ints([]), none) == 0
    assert kerr_attn.fwd_cached(ctx, cache, q, q, lse, ints([0]), ints([]), none, 1) == 0
