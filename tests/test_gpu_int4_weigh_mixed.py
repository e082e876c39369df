"""GPU: attention weight from queries of very different sizes in one call.

bf16 queries span 2^254, and each counts by its own size: one that is large must not cost its neighbours their bits.  The
tolerance is that of test_gpu_int4_weigh.py, relative to each query's own largest element.  Queries of 1e9 and more get
an lse far above their scores (their weights are 0): fp32 does not hold the difference of two such numbers."""
import math

import pytest
import torch

from test_gpu_int4_weigh import DEV, _cache, _check, _expected, _fill, _query

pytestmark = pytest.mark.gpu

SIZES = (1.0, 1e-6, 1e9, 1e30, 0.0, 3e4)


def _mixed(c, R, Hq, M, lens, shift):
    q = _query((R, Hq, M, c.D), 11, torch.bfloat16)
    size = torch.tensor(SIZES, device=DEV)[(torch.arange(M, device=DEV)[None] + torch.arange(Hq, device=DEV)[:, None] + shift)
                                           % len(SIZES)]
    q = (q.float() * size[None, :, :, None]).bfloat16()
    lse = torch.zeros(R, Hq, M, device=DEV)
    from test_gpu_int4_weigh import _parts
    for i in range(R):
        a, b = _parts(c, 0, i)
        for h in range(Hq):
            x = q[i, h].double() @ (a + b)[h // (Hq // c.H)].T * c.D ** -0.5
            see = torch.arange(lens[i], device=DEV)[None] <= (lens[i] - M + torch.arange(M, device=DEV))[:, None]
            l = torch.logsumexp(torch.where(see, x, -math.inf), -1)
            far = size[h] > 1e3
            lse[i, h] = torch.where(far, 2 * x.abs().amax(-1) + 1e3, l).float()
    return q, lse


@pytest.mark.parametrize("dim,group", [(64, 64), (64, 16), (128, 128), (128, 64), (128, 32), (256, 256), (256, 64)])
@pytest.mark.parametrize("M,rep", [(8, 1), (4, 4), (11, 3), (40, 3), (150, 1)])
def test_each_query_by_its_own_size(dim, group, M, rep):
    c = _cache(heads=2, dim=dim, group=group)
    lens = [M + 200, M, M + 33]
    _fill(c, lens, seed=dim + group)
    for shift in (0, 3):
        q, lse = _mixed(c, 3, 2 * rep, M, lens, shift)
        c.weights.zero_()
        c.weigh(0, q, lse)
        c.check()
        assert torch.isfinite(c.weights).all()
        _check(c, torch.zeros_like(c.weights), _expected(c, 0, q, lse, [0, 1, 2], [M] * 3))


@pytest.mark.parametrize("columns", [16, 33, 130])
def test_one_large_query_changes_no_other(columns):
    """The same call without the large query: what is left has the same bits, whichever kernel it is."""
    c = _cache(heads=1)
    _fill(c, [300], seed=1)
    q = _query((1, 1, columns, 128), 5, torch.bfloat16)
    lse = torch.full((1, 1, columns), 6.0, device=DEV)
    lse[0, 0, 7] = float("inf")                              # counts for nothing, whatever its size
    c.weigh(0, q, lse)
    want = c.weights.clone()
    for size in (1e-20, 1e12, 2e37):
        big = q.clone()
        big[0, 0, 7] = (q[0, 0, 7].float().sign() * size).bfloat16()
        c.weights.zero_()
        c.weigh(0, big, lse)
        c.check()
        assert torch.equal(c.weights, want)
