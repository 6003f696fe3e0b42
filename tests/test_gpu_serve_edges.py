"""GPU tests of the serving calls at their edges: offsets that do not ascend, waits
that run out, weights and values far below the largest.  Against serve_ref's 64-bit forms."""
import math

import pytest
import torch

import kerr_attn
import serve_ref
from test_gpu_serve import ints, randn

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
