"""GPU: queries that are not finite, in attention over the 4-bit cache.

A query with NaN or an infinity has no softmax: its output row and its lse are NaN, and the other rows of the call
are what they are without it.  A query that sees no token is answered without it: a zero row, lse -inf.

The other rows' bits may change (the rows of a tile move their maxima together), so both calls are within the
rounding of the exact result: 2^-11 (fp16) or 2^-8 (bf16) of it each, and twice as much together; the weights' and
values' own roundings, 2^-11 of the largest value each at most, likewise.
"""
import math

import pytest
import torch

import test_gpu_int4_cache as base

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _others(out, lse, good, lgood, hit, vmax):
    eps = 2.0 ** -11 if out.dtype == torch.float16 else 2.0 ** -8
    a, b = out[~hit].double(), good[~hit].double()
    assert ((a - b).abs() <= 2 * eps * b.abs() + 4 * 2.0 ** -11 * vmax).all()
    assert ((lse[~hit] - lgood[~hit]).abs() <= 2.0 ** -19 * lgood[~hit].abs() + 2e-5).all()


@pytest.mark.parametrize("dim,group,dtype", [(64, 64, torch.float16), (128, 128, torch.float16),
                                             (128, 32, torch.bfloat16), (256, 64, torch.float16),
                                             (256, 128, torch.bfloat16)])
@pytest.mark.parametrize("rep,m", [(1, 1), (4, 1), (7, 1), (8, 4)])
@pytest.mark.parametrize("lens", [[5, 300, 33], [3000, 5000, 70]])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_query_that_is_not_finite(dim, group, dtype, rep, m, lens, bad):
    c = base._filled(lens, dim, group)
    q = base._rand((3, 2 * rep, m, dim), 5, dtype)
    good, lgood = c.attend(0, q, return_lse=True)
    odd = q.clone()
    hit = torch.zeros(3, 2 * rep, m, dtype=torch.bool, device=DEV)
    for i, h, j, d in ((0, 0, 0, 0), (1, rep, m - 1, dim - 1), (2, 2 * rep - 1, 0, 7)):
        odd[i, h, j, d] = bad
        hit[i, h, j] = True
    out, lse = c.attend(0, odd, return_lse=True)
    c.check()
    assert torch.isnan(out[hit]).all() and torch.isnan(lse[hit]).all()
    _others(out, lse, good, lgood, hit, float(base._reference(c, 0, q[:, :, :0], [0, 1, 2], [0] * 3, 1)[2].max()))


def test_units_merged_by_the_second_kernel():
    """A table so long that the parts of a unit are merged by a launch of their own."""
    c = base._cache(1, 300, 1, 128, 64, 2, 4096)
    k = base._rand((2, 1, 4000, 128), 6, torch.float16)
    c.append(0, k, k, None, c.reserve(None, 4000))
    q = base._rand((2, 4, 3, 128), 7, torch.float16)
    good, lgood = c.attend(0, q, return_lse=True)
    odd = q.clone()
    odd[1, 2, 1, 100] = math.nan
    out, lse = c.attend(0, odd, return_lse=True)
    c.check()
    hit = torch.zeros(2, 4, 3, dtype=torch.bool, device=DEV)
    hit[1, 2, 1] = True
    assert torch.isnan(out[hit]).all() and torch.isnan(lse[hit]).all()
    _others(out, lse, good, lgood, hit, float(base._reference(c, 0, q[:, :, :0], [0, 1], [0] * 2, 1)[2].max()))


def test_one_that_sees_nothing():
    """No token, queries before the row's first token, and queries past n_new."""
    c = base._filled([0, 1, 40], 128, 128)
    q = base._rand((3, 4, 3, 128), 8, torch.float16)
    q[0, :, 0, 0] = math.nan
    q[1, :, 0, 0] = math.nan
    q[1, 0, 2, 0] = math.inf
    q[2, :, 2, 5] = -math.inf
    n = torch.tensor([3, 3, 2], dtype=torch.int32, device=DEV)
    out, lse = c.attend(0, q, n_new=n, return_lse=True)
    c.check()
    for i, j in ((0, 0), (0, 1), (0, 2), (1, 0), (1, 1), (2, 2)):
        assert (out[i, :, j] == 0).all() and (lse[i, :, j] == -math.inf).all()
    assert torch.isnan(out[1, 0, 2]).all() and torch.isnan(lse[1, 0, 2])
    assert torch.isfinite(out[1, 1:, 2]).all() and torch.isfinite(out[2, :, :2]).all()
