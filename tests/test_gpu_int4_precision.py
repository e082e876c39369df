"""GPU: attention over the 4-bit cache is as exact as its output's type, whatever the weights' spread.

Measure: the root mean square of (output - formula in 64 bits) over the one of (formula rounded to the output's type -
formula), row by row of the call.  Bound, derived before the first run: 1.1.  The kernel's own error has to stay below
sqrt(1.1^2 - 1) = 0.46 of the output's rounding, some 1.6e-4 (fp16: 2.1e-4 / 2 of the row's root mean square; bf16:
1.66e-3).  An fp16 output's weights carry 22 bits, its sums 24: some 1e-6.  A bf16 output's weights and values are
rounded to fp16 once each, 2^-12 root mean square at most: 3.5e-4.
"""
import math

import pytest
import torch

import test_gpu_int4_cache as base

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _fields(c, rows):
    """K and V values (row, head, token, channel) in 64 bits of rows that all hold the same number of tokens."""
    n = int(c.lens[rows[0]])
    rec = c.buf[0, c.table[rows, :(n + 31) // 32].long()].transpose(1, 2)          # (row, H, blocks, rec)
    L, G, out = c.layout, c.layout.n_groups, []
    for co, po in ((L.kc, L.kp), (L.vc, L.vp)):
        b = rec[..., co:co + 16 * c.D].reshape(len(rows), c.H, -1, c.D // 2)[:, :, :n]
        p = rec[..., po:po + 128 * G].contiguous().view(torch.float16).reshape(len(rows), c.H, -1, G, 2)[:, :, :n]
        code = torch.stack([b >> 4, b & 15], -1).flatten(-2).double().unflatten(-1, (G, -1))
        out.append((code * p[..., :1].double() + p[..., 1:].double()).flatten(-2))
    return out


def _formula(k, v, q):
    """softmax(q k^T / sqrt(D)) v in 64 bits, causal for the M newest tokens; also the first token's weights."""
    R, Hq, M, D = q.shape
    rep = Hq // k.shape[1]
    x = torch.einsum("rhemd,rhtd->rhemt", q.double().unflatten(1, (-1, rep)), k) / math.sqrt(D)
    t, n = torch.arange(k.shape[2], device=DEV), k.shape[2]
    x.masked_fill_(t > (n - M + torch.arange(M, device=DEV))[:, None], -math.inf)
    w = torch.softmax(x, -1)
    return torch.einsum("rhemt,rhtd->rhemd", w, v).flatten(1, 2), w[..., 0]


def _ratio(got, ref):
    """Root mean square errors: the kernel's over that of the formula rounded once; the worst row."""
    own = (ref.to(got.dtype).double() - ref).square().flatten(1).mean(1).sqrt()
    return float(((got.double() - ref).square().flatten(1).mean(1).sqrt() / own).max())


def _one_prompt(share, own_value, hq, m, dtype):
    """75 rows of 8 heads that share one prompt of 32K tokens, so that a unit is hardly cut; `share` of the weight is
    on the first token, whose value is 0 or of the others' size.  The worst row's ratio."""
    import akv
    n, rows = 32768, 75
    c = akv.Int4PagedCache(1, 1040, 8, 128, max_seqs=rows, max_blocks=1025, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(5)
    k = torch.randn(1, 8, n, 128, generator=g, device=DEV) * 1.2
    v = torch.randn(1, 8, n, 128, generator=g, device=DEV) * 30     # outputs in fp16's normal range
    if not own_value:
        v[:, :, 0] = 0
    k[:, :, 0] = 0
    k[..., 0] = 0
    # channel 0 of every query is 8 and of every other key 0: the first token's logit is 8 k / sqrt(128)
    if share:
        k[:, :, 0, 0] = (math.log(n) + 0.72 + math.log(share / (1 - share))) * math.sqrt(128) / 8
    c.append(0, k.half(), v.half(), [0], c.reserve([0], n))
    c.fork(torch.zeros(rows - 1, dtype=torch.int32, device=DEV), torch.arange(1, rows, dtype=torch.int32, device=DEV))
    q = torch.randn(rows, hq, m, 128, generator=g, device=DEV).to(dtype)
    q[..., 0] = 8
    out = c.attend(0, q)
    c.check()
    K, V = _fields(c, [0])
    worst = 0.0
    for i in range(0, rows, 5):
        ref, first = _formula(K, V, q[i:i + 1])
        worst = max(worst, _ratio(out[i:i + 1], ref))
    if share:
        assert abs(float(first.mean()) - share) < 0.1
    return worst


@pytest.mark.parametrize("hq,m,dtype", [(32, 1, torch.float16), (64, 1, torch.float16), (32, 4, torch.float16),
                                        (64, 1, torch.bfloat16)])
def test_sums_over_many_tokens(hq, m, dtype):
    assert _one_prompt(0.0, True, hq, m, dtype) <= 1.1


@pytest.mark.parametrize("share", [0.5, 0.9, 0.99])
@pytest.mark.parametrize("own_value", [True, False])
@pytest.mark.parametrize("hq,m,dtype", [(32, 1, torch.float16), (64, 1, torch.float16), (32, 4, torch.float16),
                                        (64, 1, torch.bfloat16)])
def test_most_of_the_weight_on_the_first_token(share, own_value, hq, m, dtype):
    """The other tokens' weights, each a 32768th of what is left, still make the output as exact as its type."""
    assert _one_prompt(share, own_value, hq, m, dtype) <= 1.1


@pytest.mark.parametrize("dim,group", [(64, 64), (64, 32), (64, 16), (128, 128), (128, 64), (128, 32),
                                       (256, 256), (256, 128), (256, 64)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rep,m", [(1, 1), (4, 1), (7, 1), (4, 3), (8, 4)])
def test_every_shape(dim, group, dtype, rep, m):
    """Long rows, cut over many CTAs; unit normal values."""
    c = base._cache(1, 200, 2, dim, group, 2, 98)
    g = torch.Generator(device=DEV).manual_seed(dim + group)
    k, v = (torch.randn(2, 2, 3001, dim, generator=g, device=DEV).half() for _ in range(2))
    c.append(0, k, v, None, c.reserve(None, 3001))
    q = torch.randn(2, 2 * rep, m, dim, generator=g, device=DEV).to(dtype)
    out = c.attend(0, q)
    c.check()
    assert _ratio(out, _formula(*_fields(c, [0, 1]), q)[0]) <= 1.1


@pytest.mark.parametrize("dim,group,dtype", [(64, 64, torch.float16), (128, 128, torch.float16),
                                             (128, 32, torch.float16), (256, 128, torch.float16),
                                             (128, 128, torch.bfloat16), (128, 32, torch.bfloat16)])
@pytest.mark.parametrize("rep,m,where", [(4, 1, "light"), (8, 1, "light"), (4, 4, "light"), (4, 4, "unseen")])
def test_one_token_of_much_larger_values(dim, group, dtype, rep, m, where):
    """A token whose values are 3,000 times the others' and that hardly counts, or is the last new one."""
    n = 1111
    c = base._cache(1, 80, 2, dim, group, 2, 36)
    g = torch.Generator(device=DEV).manual_seed(dim + group + m)
    k, v = (torch.randn(2, 2, n, dim, generator=g, device=DEV) for _ in range(2))
    q = torch.randn(2, 2 * rep, m, dim, generator=g, device=DEV)
    v *= 0.01
    q[..., 0], k[..., 0] = 4, 0
    at = n - 1 if where == "unseen" else 500
    v[:, :, at] *= 3000
    if where == "light":
        k[:, :, at] = 0
        k[:, :, at, 0] = -20 * math.sqrt(dim) / 4            # its logit: -20
    c.append(0, k.half(), v.half(), None, c.reserve(None, n))
    q = q.to(dtype)
    out = c.attend(0, q)
    c.check()
    ref = _formula(*_fields(c, [0, 1]), q)[0]
    if where == "unseen":
        out, ref = out[:, :, :-1], ref[:, :, :-1]
    assert _ratio(out, ref) <= 1.1
