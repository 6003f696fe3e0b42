"""Plain 64-bit forms of the serving calls (kattn_fwd_packed, kattn_cache_*,
kattn_fwd_cached) on the CPU, with bounds on how far a kernel may be off.

Bounds.  With u = eps/2 of a type (half a step: f32 2^-24, f16 2^-11, bf16
2^-8), a row's scores s_j, weights p_j (sum one) and A = sum_j p_j |v_j|:

- A score is off by at most D = c_s * |scale| * max_j sum_i |q_i k_ji|, where
  c_s = 3 * 2^-22 for f32 (products of f16 hi + lo pairs, 11 bits each: each
  operand is off by 2^-22 of itself and lo * lo, 2^-22, is left out) plus the f32 sums'
  (d + 3) * 2^-24, which stand alone for 16-bit types, whose products are exact.
  Pairs stand behind a power of two that brings the largest of a row or of some
  keys to 2^14 or above; below 2^-3 the lo loses up to 2^-25, so an element is off
  by 2^-39 of the largest besides: a score by |scale| * 2 * d * 2^-39 max|q| max|k|.
- Weights change by a factor within exp(+-2 D), exp2's own 2^-21 included by
  adding it to D: o moves by at most 2 D A.
- Weights enter the second product rounded: by u of the type for 16-bit types
  (c_v = u; the unnormalised weights, at most 2^8, lose at most 2^-24 below
  f16's normal range, and there are `keys` of them: keys * 2^-24 * max|v|),
  by 3 * 2^-22 for f32, where a weight, held times 2^7 and at least one for some key,
  is off by 2^-32 besides, and v by 2^-37 of the largest (its power of two is kept for
  keys up to four times the first): (keys * 2^-32 + 2^-37) * max|v|; its f32 sums and the division add (keys + 8) * 2^-24.
- The output is rounded once: u |o|.
- lse is off by D, by 2^-21 for the logarithm, and by its rounding, 2^-23 |lse|.
"""
import math

import torch

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LIMIT = {0: 127.0, 1: 448.0}


def attend(q, k, v, seen, scale, dtype):
    """q [t, H, d], k, v [l, Hkv, d] (64 bits), seen [t, l]: o [t, H, d], lse
    [H, t] and their bounds."""
    t, H, d = q.shape
    length, group = k.shape[0], H // k.shape[1] if k.shape[1] else 1
    kh, vh = (x.repeat_interleave(group, 1).transpose(0, 1) for x in (k, v))  # [H, l, d]
    qh = q.transpose(0, 1)
    if length == 0:
        z = torch.zeros(t, H, d, dtype=torch.float64)
        return z, torch.full((H, t), -math.inf, dtype=torch.float64), z, torch.zeros(H, t, dtype=torch.float64)
    s = (qh @ kh.mT) * scale
    s = torch.where(seen, s, torch.full((), -math.inf, dtype=s.dtype))
    lse = torch.logsumexp(s, -1)
    some = lse > -math.inf
    p = torch.where(seen & some[..., None], torch.exp(s - torch.where(some, lse, 0.0)[..., None]), 0.0)
    vz = torch.where(seen.any(0)[:, None], vh, torch.zeros_like(vh))  # rows that nobody sees do not count
    o = p @ vz
    A = p @ vz.abs()
    u = U[dtype]
    c_s = (3 * 2.0 ** -22 if dtype == torch.float32 else 0.0) + (d + 3) * 2.0 ** -24
    most = torch.where(seen, (qh.abs() @ kh.abs().mT) * abs(scale), 0.0).amax(-1)
    D = c_s * most + 2.0 ** -21
    if dtype == torch.float32:
        D = D + abs(scale) * 2 * d * 2.0 ** -39 * qh.abs().amax(-1) * kh.abs().amax((1, 2))[:, None]
    c_v = 3 * 2.0 ** -22 if dtype == torch.float32 else u
    low = (length * 2.0 ** -32 + 2.0 ** -37 if dtype == torch.float32 else length * 2.0 ** -24) * \
        vz.abs().amax((1, 2))[:, None, None]
    bo = A * (2 * D[..., None] + c_v + (length + 8) * 2.0 ** -24) + low + u * o.abs() + 1e-30
    bl = D + 2.0 ** -21 + 2.0 ** -23 * torch.where(some, lse, 0.0).abs()
    return o.transpose(0, 1), lse, bo.transpose(0, 1), bl


def packed(q, k, v, cu_q, cu_k, H, Hkv, causal, scale):
    """kattn_fwd_packed on packed rows; rows of no sequence are NaN."""
    dtype, d = q.dtype, q.shape[1] // H
    q, k, v = (x.cpu().double() for x in (q, k, v))
    N = q.shape[0]
    o, bo = (torch.full((N, H, d), math.nan, dtype=torch.float64) for _ in range(2))
    lse, bl = (torch.full((H, N), math.nan, dtype=torch.float64) for _ in range(2))
    for s in range(len(cu_q) - 1):
        a, b, c, e = cu_q[s], cu_q[s + 1], cu_k[s], cu_k[s + 1]
        nq, nk = b - a, e - c
        seen = torch.ones(nq, nk, dtype=torch.bool)
        if causal:
            seen = torch.arange(nk) <= torch.arange(nq)[:, None] + nk - nq
        r = attend(q[a:b].view(nq, H, d), k[c:e].view(nk, Hkv, d), v[c:e].view(nk, Hkv, d), seen, scale, dtype)
        o[a:b], lse[:, a:b], bo[a:b], bl[:, a:b] = r
    return o.view(N, H * d), lse, bo.view(N, H * d), bl


def quantise(x, fmt):
    """Codes (as their 64-bit values) and f32 scales of rows along the last dimension."""
    x = x.cpu().float()
    m = x.abs().amax(-1)
    usual = (m >= 2.0 ** -100) & (m < math.inf)
    limit = torch.full_like(m, LIMIT[fmt])
    inverse = torch.where(usual, limit / m, 0.0)
    scale = torch.where(usual, m / limit, torch.where(m < 2.0 ** -100, 0.0, math.nan))
    y = torch.where(usual[..., None], x.double() * inverse.double()[..., None], 0.0)
    if fmt == 0:
        return torch.round(y), scale
    e = torch.frexp(y).exponent.clamp(min=-5) - 4
    step = torch.ldexp(torch.ones_like(y), e)
    return (torch.round(y / step) * step).clamp(-448, 448), scale


def values(cache):
    """The cache's codes as 64-bit values [pages, Hkv, page, d], without their scales."""
    out = []
    for c in (cache.k, cache.v):
        c = c.cpu()
        out.append(c.view(torch.int8).double() if cache.format == 0 else c.view(torch.float8_e4m3fn).double())
    return out


def position(cache, table, s, p):
    """(page, place) of position p, or None where it does not exist."""
    i = p // cache.page_size
    if p < 0 or i >= table.shape[1]:
        return None
    page = int(table[s, i])
    return (page, p % cache.page_size) if 0 <= page < cache.n_pages else None


def cached(cache, q, cu, kv_len, table, H, tree, scale):
    """kattn_fwd_cached on the cache's contents; rows of no sequence are NaN."""
    dtype, d, Hkv = q.dtype, cache.d, cache.n_kv_head
    kc, vc = values(cache)
    ks, vs = (x.cpu().double()[..., None] for x in (cache.k_scale, cache.v_scale))
    kc, vc = kc * ks, vc * vs
    table = table.cpu()
    q = q.cpu().double()
    N = q.shape[0]
    o, bo = (torch.full((N, H, d), math.nan, dtype=torch.float64) for _ in range(2))
    lse, bl = (torch.full((H, N), math.nan, dtype=torch.float64) for _ in range(2))
    for s, length in enumerate(kv_len):
        a, b = cu[s], cu[s + 1]
        n = b - a
        if n == 0:
            continue
        at, cols = [], []
        for p in range(max(length, 0)):
            w = position(cache, table, s, p)
            if w is None:
                continue
            j = p - (length - n)
            if j < 0:
                cols.append([True] * n)
            elif tree is None:
                cols.append([j <= i for i in range(n)])
            else:
                cols.append([j < 64 and bool((int(tree[a + i]) >> j) & 1) for i in range(n)])
            at.append(w)
        pages, places = [w[0] for w in at], [w[1] for w in at]
        seen = torch.tensor(cols, dtype=torch.bool).view(len(at), n).T
        k, v = kc[pages, :, places].view(-1, Hkv, d), vc[pages, :, places].view(-1, Hkv, d)
        r = attend(q[a:b].view(n, H, d), k, v, seen, scale, dtype)
        o[a:b], lse[:, a:b], bo[a:b], bl[:, a:b] = r
    return o.view(N, H * d), lse, bo.view(N, H * d), bl


def check(got, want, bound, what):
    """Every element within its bound; the same infinities; NaN in `want`: not looked at."""
    got = got.cpu().double()
    look = ~torch.isnan(want)
    inf = torch.isinf(want) & look
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities differ"
    look &= ~inf
    off = (got - want).abs()
    bad = look & ~(off <= bound)
    if bad.any():
        i = int(torch.where(bad, off / bound, 0.0).nan_to_num(1e30).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {int(look.sum())} out of bounds, worst at {i}: got "
                             f"{got.flatten()[i]}, want {want.flatten()[i]} +- {bound.flatten()[i]}")
