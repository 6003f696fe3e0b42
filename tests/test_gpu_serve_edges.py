"""GPU tests of the serving calls at their edges: offsets that do not ascend, waits
that run out, weights and values far below the largest.  Against serve_ref's 64-bit forms."""
import math

import pytest
import torch

import kerr_attn
import serve_ref
from test_gpu_serve import fill, ints, make_cache, offsets, randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = kerr_attn.Context(0)
    yield c
    c.check_device()
    c.close()


def test_packed_plan_ends_inside_a_sequence(ctx):
    # Overlapping offsets make 513 items a key head, one more than the plan of a line takes, so that a head ends inside
    # the last sequence: the walk goes on with the next head's first, not with what lies behind the offsets (here
    # a sequence of rows that nobody owns).
    gen = torch.Generator().manual_seed(31)
    H, Hkv, d, M, N = 12, 3, 64, 1728, 1792
    q = randn(gen, N, H * d, dtype=torch.bfloat16)
    k, v = (torch.zeros(300000, Hkv * d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    for x in (k, v):
        x[:N] = randn(gen, N, Hkv * d, dtype=torch.bfloat16)
    offsets_ = ints([0, M] * 19 + [N])
    o, lse = torch.full_like(q, 7.0), torch.full((H, N), 7.0, device="cuda")
    assert kerr_attn.fwd_packed(ctx, q, k, v, o, lse, offsets_[:-1], offsets_[:-1], H, Hkv) == 2
    assert (o[M:] == 7).all() and (lse[:, M:] == 7).all()
    want, wl, bo, bl = serve_ref.packed(q[:M], k[:M], v[:M], [0, M], [0, M], H, Hkv, True, 1 / math.sqrt(d))
    serve_ref.check(o[:M], want, bo, "o")
    serve_ref.check(lse[:, :M], wl, bl, "lse")


def check_withheld(call, limit_ns):
    """call(ctx) with a copy withheld: the waits run out after the limit, the call ends with the status word set,
    and the same context then gives the same bits as before."""
    with kerr_attn.Context(0) as ctx:
        usual = [x.clone() for x in call(ctx)]
        ctx.check_device()
        for _ in range(3):
            ctx.set_wait_limit(limit_ns)
            ctx.test_withhold_next_load()
            call(ctx)
            with pytest.raises(kerr_attn.KattnError) as e:
                ctx.check_device()
            assert e.value.status == kerr_attn.KATTN_ERR_DEVICE_TIMEOUT
            ctx.check_device()  # the report cleared the flag
            ctx.set_wait_limit(0)
            again = call(ctx)
            ctx.check_device()
            assert all(torch.equal(a, b) for a, b in zip(usual, again))


def packed_call(dtype, d, whole):
    gen = torch.Generator().manual_seed(41)
    nq, H, Hkv = [300, 1, 777, 40, 1200], 32 if whole else 8, 16 if whole else 4
    nk = nq if whole else [900, 2, 4777, 1600, 1200]
    q = randn(gen, sum(nq), H * d, dtype=dtype)
    k, v = (randn(gen, sum(nk), Hkv * d, dtype=dtype) for _ in range(2))
    cu_q, cu_k = ints(offsets(nq)), ints(offsets(nk))
    o, lse = torch.empty_like(q), torch.empty(H, q.shape[0], device="cuda")

    def call(ctx):
        # Whole items, or parts and a join.
        assert kerr_attn.fwd_packed(ctx, q, k, v, o, lse, cu_q, cu_k, H, Hkv) == (1 if whole else 2)
        return o, lse

    return call


def cached_call(dtype, d, fmt, rows):
    gen = torch.Generator().manual_seed(42)
    kv_len, new, Hkv = [5000, 300, 9000, 40], [rows, 1, 1, rows], 8
    cache, table = make_cache(kv_len, 32, Hkv, d, fmt, seed=43)
    with kerr_attn.Context(0) as ctx:
        fill(ctx, cache, table, kv_len, dtype, seed=44)
    H = 2 * Hkv
    q = randn(gen, sum(new), H * d, dtype=dtype)
    cu, lengths = ints(offsets(new)), ints(kv_len)
    o, lse = torch.empty_like(q), torch.empty(H, q.shape[0], device="cuda")

    def call(ctx):
        kerr_attn.fwd_cached(ctx, cache, q, o, lse, cu, lengths, table, H)
        return o, lse

    return call


MS = 1_000_000


@pytest.mark.parametrize("whole", [True, False])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_packed_withheld_copy(dtype, d, whole):
    check_withheld(packed_call(dtype, d, whole), MS)


@pytest.mark.parametrize("rows", [1, 30])
@pytest.mark.parametrize("fmt", [kerr_attn.CACHE_INT8, kerr_attn.CACHE_E4M3])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_cached_withheld_copy(dtype, d, fmt, rows):
    check_withheld(cached_call(dtype, d, fmt, rows), MS)


@pytest.mark.parametrize("whole", [True, False])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_packed_withheld_copy_f32(d, whole):
    # The four warps that convert f32 tiles meet at every tile: all of them leave when one gives up.
    check_withheld(packed_call(torch.float32, d, whole), MS)


@pytest.mark.parametrize("whole", [True, False])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_packed_gives_up_with_copies_in_flight(dtype, d, whole):
    # Waits run out at their first look, each warp where it happens to be, while the copies behind the withheld one are
    # on their way: they land before the shared memory is released.
    check_withheld(packed_call(dtype, d, whole), 1)


@pytest.mark.parametrize("rows", [1, 30])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_cached_gives_up_with_copies_in_flight(dtype, d, rows):
    check_withheld(cached_call(dtype, d, kerr_attn.CACHE_INT8, rows), 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_packed_many_small_weights(ctx, dtype):
    # One key takes nearly all of the weight and has a value of zero: the output is 60000 others', each 2^-26 of it.
    # As many rows as whole items take, so that every item sees all keys; all rows are alike.
    d, rows, n = 64, 115200, 60000
    q = torch.zeros(rows, d, dtype=dtype, device="cuda")
    q[:, 0] = 4.0
    k = torch.zeros(n + 1, d, dtype=dtype, device="cuda")
    k[1:, 0] = -4.5
    v = torch.rand(n + 1, d, generator=torch.Generator().manual_seed(45)).add(0.5).to(dtype).cuda()
    v[0] = 0
    o, lse = torch.empty_like(q), torch.empty(1, rows, device="cuda")
    assert kerr_attn.fwd_packed(ctx, q, k, v, o, lse, ints([0, rows]), ints([0, n + 1]), 1, 1, causal=False, scale=1.0) == 1
    w = math.exp(-18.0)
    want = w * v[1:].double().sum(0) / (1 + n * w)
    # A weight, held times 2^7, is off by 2^-25 where f16 is subnormal, else by u of itself; the output by u; the score by
    # its product's f32 sums and exp2's 2^-21; O's sums of 16 keys at a time, and l's of 128, by an f32 step each.
    u = serve_ref.U[dtype]
    relative = 2 * u + 2 * ((d + 3) * 2.0 ** -24 * 18 + 2.0 ** -21) + (n / 16) * 2.0 ** -23 + (n / 128) * 2.0 ** -24
    bound = n * 2.0 ** -32 * v.double().max() + relative * want
    assert ((o.double() - want).abs() <= bound).all()
    assert (lse - math.log1p(n * w)).abs().max() <= 2.0 ** -20 + (n / 128) * 2.0 ** -24


@pytest.mark.parametrize("power", [0, 10, 20, 30])
@pytest.mark.parametrize("fmt", [kerr_attn.CACHE_INT8, kerr_attn.CACHE_E4M3])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_cached_beside_a_far_larger_value(ctx, dtype, fmt, power):
    # A drafted token whose values are 2^power times the others', which only the second row sees: the first row's
    # positions are off by 2^-31 of the largest value each, besides the usual bounds.
    gen = torch.Generator().manual_seed(46)
    H, Hkv, d, length = 4, 2, 64, 6
    cache, table = make_cache([length], 16, Hkv, d, fmt, seed=47)
    k, v = randn(gen, length, Hkv * d), randn(gen, length, Hkv * d)
    v[length - 1] *= 2.0 ** power
    kerr_attn.cache_append(ctx, cache, k, v, ints([0, length]), ints([length]), table)
    q = randn(gen, 2, H * d, dtype=dtype)
    o, lse = torch.empty_like(q), torch.empty(H, 2, device="cuda")
    kerr_attn.fwd_cached(ctx, cache, q, o, lse, ints([0, 2]), ints([length]), table, H, tree=torch.tensor([1, 3]).cuda())
    kc, vc = serve_ref.values(cache)
    page = int(table[0, 0])
    held = [(c * s.cpu().double()[..., None])[page].transpose(0, 1) for c, s in ((kc, cache.k_scale), (vc, cache.v_scale))]
    for row, n in ((0, length - 1), (1, length)):
        want, wl, bo, bl = serve_ref.attend(q[row:row + 1].cpu().double().view(1, H, d), held[0][:n], held[1][:n],
                                            torch.ones(1, n, dtype=torch.bool), 1 / math.sqrt(d), dtype)
        bo = bo + n * 2.0 ** -31 * held[1].abs().max()
        if dtype == torch.float16:  # from 65520 on the nearest f16 is an infinity; within the bound of it either is right
            want = torch.where(want.abs() - bo > 65520, want * math.inf, want)
            want = torch.where((want.abs() - 65520).abs() <= bo, math.nan, want)
        serve_ref.check(o[row:row + 1].view(1, H, d), want, bo, f"o of row {row}")
        serve_ref.check(lse[:, row:row + 1], wl, bl, f"lse of row {row}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_cached_shared_pages(ctx, dtype):
    # Two sequences whose earlier positions lie on the same pages, and one that has a page twice.
    H, Hkv, d, page = 4, 2, 64, 16
    cache, _ = make_cache([160], page, Hkv, d, kerr_attn.CACHE_INT8, seed=48)
    table = ints([[3, 5, 1, 7], [3, 5, 2, 0], [4, 4, 6, 0]])
    gen = torch.Generator().manual_seed(49)
    cu, kv_len = [0, 50, 53, 56], [50, 35, 40]
    k, v = randn(gen, 56, Hkv * d, dtype=dtype), randn(gen, 56, Hkv * d, dtype=dtype)
    for s in range(3):  # one after the other: the third's pages hold what is on them
        kerr_attn.cache_append(ctx, cache, k[cu[s]:cu[s + 1]], v[cu[s]:cu[s + 1]], ints([0, cu[s + 1] - cu[s]]),
                               ints(kv_len[s:s + 1]), table[s:s + 1])
    q = randn(gen, 7, H * d, dtype=dtype)
    o, lse = torch.empty_like(q), torch.empty(H, 7, device="cuda")
    kerr_attn.fwd_cached(ctx, cache, q, o, lse, ints([0, 1, 4, 7]), ints(kv_len), table, H)
    want, wl, bo, bl = serve_ref.cached(cache, q, [0, 1, 4, 7], kv_len, table, H, None, 1 / math.sqrt(d))
    serve_ref.check(o, want, bo, "o")
    serve_ref.check(lse, wl, bl, "lse")


def test_cached_broken_offsets_and_lengths_stay_inside(ctx):
    # Offsets that descend or leave the arrays, lengths below zero and past the table, pages that do not exist: every
    # call keeps inside its arrays.
    H, Hkv, d, N, page = 4, 2, 64, 100, 16
    cu, kv_len = ints([0, 500, 40, -7, 1000, 60, 100]), ints([-5, 2 ** 31 - 1, 33, 90, 0, 64])
    table = ints([[0, 9, -3, 2, 2 ** 31 - 1, 1]] * 6)
    guard = torch.full((2, 6, Hkv, page, d), 5, dtype=torch.int8, device="cuda")
    scales = torch.full((2, 6, Hkv, page), 3.0, device="cuda")
    cache = kerr_attn.KVCache(guard[0, 1:4], guard[1, 1:4], scales[0, 1:4], scales[1, 1:4])  # pages amid others
    wide = torch.full((4, N + 40, H * d), 3.0, device="cuda")
    q, o, k, v = (x[20:20 + N] for x in wide)
    lse = torch.zeros(H, N, device="cuda")
    kv = [x[:, :Hkv * d] for x in (k, v)]
    kerr_attn.cache_append(ctx, cache, *kv, cu, kv_len, table)
    kerr_attn.cache_read(ctx, cache, *kv, cu, kv_len, table)
    kerr_attn.fwd_cached(ctx, cache, q, o, lse, cu, kv_len, table, H)
    ctx.check_device()
    assert (wide[:, :20] == 3).all() and (wide[:, 20 + N:] == 3).all() and (wide[2:, :, Hkv * d:] == 3).all()
    for x, value in ((guard, 5), (scales, 3)):
        assert (x[:, 0] == value).all() and (x[:, 4:] == value).all()
