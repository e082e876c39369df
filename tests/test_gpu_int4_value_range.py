"""GPU: attention over V values at the ends of fp16's range.

append holds infinities and bf16 values past fp16's range to +-65504, and a group's scale is rounded to fp16, so 15
steps of it (or none, with scale and zero taken together) can lie past the largest fp16 by up to 15 halves of the
scale's last place: 30 at 65504.  Such a value may be held to 65504, as ``read`` does; it may not become infinite,
because a token that a query does not see has weight 0, and 0 times infinity is NaN.

Bounds, derived before the first run.  Where values are unpacked with scale and zero (four groups, or two and more
than eight query rows a KV head), a query that does not see such a token gives the same bits as over a cache where
that token is an ordinary one: the weights and values of the others are the same numbers.  One that sees it: a value
is off by two fp16 roundings (16 each at 65504), or by 30 where it is held, at most 2^-10 of 65504; one fp16
rounding of the weight, 2^-11; the output's own, 2^-8.  With out = sum w v and sum w = 1 the error is at most
(2^-10 + 2^-11 + 2^-20) max|v| + 2^-8 |out|.
"""
import pytest
import torch

import test_gpu_int4_cache as base

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _edge_rows(kind, shape, dtype):
    """One token's V rows whose groups reach past the largest fp16 in the way `kind` names."""
    x = base._rand(shape, 3, dtype)
    if kind == "inf":                     # from 0 to +inf: scale 4368, 15 steps 65520
        x = x.abs()
        x[..., 1::4], x[..., 0::4] = float("inf"), 0.0
    elif kind == "both":                  # -inf to +inf: scale 8736
        x[..., 1::4], x[..., 0::4] = float("inf"), -float("inf")
    elif kind == "large":                 # bf16 past fp16's range
        x = x.abs()
        x[..., 1::4], x[..., 0::4] = 1e5, -3.0
    else:                                 # zero -65504, scale 4086: the zero code's value rounds down past the range
        x[..., 0::4], x[..., 1::4] = -float("inf"), -4216.0
        x[..., 2::4], x[..., 3::4] = -30000.0, -50000.0
    return x.to(dtype)


@pytest.mark.parametrize("dim,group,heads_q,m", [(64, 16, 2, 3), (64, 32, 8, 4), (128, 32, 8, 5), (128, 32, 2, 2),
                                                 (128, 64, 8, 5), (256, 64, 4, 3), (256, 128, 8, 5),
                                                 (128, 128, 8, 5), (128, 64, 2, 1)])
@pytest.mark.parametrize("kind", ["inf", "both", "large", "low"])
@pytest.mark.parametrize("n", [0, 29, 1500])
def test_a_later_draft_at_the_ends_of_the_range(dim, group, heads_q, m, kind, n):
    """The last of m new tokens has V at the ends of the range: the queries before it do not see it."""
    dtype = torch.bfloat16
    edge, plain = (base._filled([n, 40], dim, group) for _ in range(2))
    k, v = base._rand((2, 2, m, dim), 1, dtype), base._rand((2, 2, m, dim), 2, dtype)
    q = base._rand((2, 2 * heads_q, m, dim), 4, dtype)
    outs = []
    for c, odd in ((edge, True), (plain, False)):
        c.buf.copy_(plain.buf)
        vv = v.clone()
        if odd:
            vv[:, :, -1] = _edge_rows(kind, (2, 2, dim), dtype)
        # room for the new tokens: one block more than the rows of _filled always have
        g = c.reserve(None, m)
        assert g.tolist() == [m, m]
        c.append(0, k, vv, None, g)
        outs.append(c.attend(0, q, None, g, return_lse=True))
        c.check()
    (a, la), (b, lb) = outs
    assert torch.isfinite(a).all()
    if dim // group * (1 if heads_q * m <= 8 else 2) >= 4:
        assert torch.equal(a[:, :, :-1], b[:, :, :-1])
    assert torch.equal(la, lb)
    ref, _, vmax, _ = base._reference(edge, 0, q, [0, 1], [m, m], dim ** -0.5)
    err = (a.double() - ref).abs()
    assert (err <= 2.0 ** -8 * ref.abs() + (2.0 ** -10 + 2.0 ** -11 + 2.0 ** -20) * vmax).all(), float(err.max())


def test_the_ends_of_the_range_in_older_tokens():
    """Tokens in whole pages, seen by every query: finite, and the values' average."""
    k, v = base._rand((1, 2, 200, 128), 5, torch.bfloat16), base._rand((1, 2, 200, 128), 6, torch.bfloat16)
    v[:, :, 40:45] = _edge_rows("inf", (1, 2, 5, 128), torch.bfloat16)
    v[:, :, 99] = _edge_rows("low", (1, 2, 128), torch.bfloat16)
    c = base._cache(1, 60, 2, 128, 32, 1, 50)
    c.append(0, k, v, None, c.reserve(None, 200))
    q = base._rand((1, 8, 5, 128), 7, torch.bfloat16)
    out = c.attend(0, q)
    c.check()
    ref, _, vmax, _ = base._reference(c, 0, q, [0], [5], 128 ** -0.5)
    assert torch.isfinite(out).all()
    err = (out.double() - ref).abs()
    assert (err <= 2.0 ** -8 * ref.abs() + (2.0 ** -10 + 2.0 ** -11 + 2.0 ** -20) * vmax).all(), float(err.max())
