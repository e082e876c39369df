"""GPU: verification of drafted tokens against exact integers (and its statistics)."""
from fractions import Fraction

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
UNIT = 1 << 40


def _units(x):
    x = np.nan_to_num(x.astype(np.float64), nan=0.0, posinf=1.0, neginf=0.0).clip(0, 1)
    return [int(v) for v in np.rint(x * UNIT)]


def _model(p, q, x, u, ul, n):
    """One sequence in exact arithmetic: (accepted, tokens)."""
    K, V = len(x), p.shape[1]
    j, out = 0, []
    while j < n:
        ok = 0 <= x[j] < V
        if ok:
            qx = Fraction(1) if q is None else Fraction(float(q[j, x[j]]))
            ok = Fraction(float(u[j])) * qx < Fraction(float(p[j, x[j]]))
        if not ok:
            break
        out.append(int(x[j]))
        j += 1
    full = _units(p[j])
    w = full
    if j < n:
        if q is None:
            w = [0 if i == x[j] else f for i, f in enumerate(full)]
        else:
            w = [max(f - g, 0) for f, g in zip(full, _units(q[j]))]
        if sum(w) == 0:
            w = full
    tot = sum(w)
    nxt = -1
    if tot:
        goal = int(float(ul) * (1 << 24)) * tot >> 24
        s = 0
        for i, f in enumerate(w):
            s += f
            if s > goal:
                nxt = i
                break
    return j, out + [nxt] + [-1] * (K - j)


def _case(B, K, V, dtype, draft, seed, sharp=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    logits = torch.randn(B, K + 1, V, generator=g, device=DEV) * sharp
    p = torch.softmax(logits, -1).to(dtype)
    q = torch.softmax(logits[:, :K] + torch.randn(B, K, V, generator=g, device=DEV) * 0.6, -1).to(dtype)
    noise = torch.rand(B, K, V, generator=g, device=DEV).clamp_min(1e-30)
    x = (q.float().log() - (-noise.log()).log()).argmax(-1) if K else torch.zeros(B, 0, dtype=torch.int64, device=DEV)
    u = torch.rand(B, K, generator=g, device=DEV)
    ul = torch.rand(B, generator=g, device=DEV)
    n = torch.randint(0, K + 1, (B,), generator=torch.Generator().manual_seed(seed)).int().to(DEV)
    return p, (q if draft else None), x, u, ul, n


def _check(p, q, x, u, ul, n=None, status=None):
    import akv
    acc, tok = akv.verify_draft(p, q, x, u, ul, n_draft=n, status=status)
    torch.cuda.synchronize()
    K = x.shape[1]
    for b in range(p.shape[0]):
        cnt = K if n is None else min(max(int(n[b]), 0), K)
        want = _model(p[b].float().cpu().numpy(), None if q is None else q[b].float().cpu().numpy(),
                      x[b].tolist(), u[b].tolist(), float(ul[b]), cnt)
        assert (int(acc[b]), tok[b].tolist()) == want, b
    return acc, tok


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (3, 2, 7), (2, 0, 100), (5, 4, 1000), (9, 3, 4097), (2, 8, 32003),
                                   (1, 40, 333), (17, 5, 128)])
def test_against_exact_integers(B, K, V, dtype, draft):
    p, q, x, u, ul, n = _case(B, K, V, dtype, draft, B * 100 + K * 10 + V)
    _check(p, q, x, u, ul, n)
    _check(p, q, x, u, ul)


def test_large_vocabulary():
    _check(*_case(3, 4, 151936, torch.float32, True, 5))


def test_edges_of_the_draw():
    """u = 0 takes the first token with weight, u just below 1 the last; equal rows, empty rows, bad values."""
    V = 5000
    p = torch.zeros(6, 2, V, device=DEV)
    q = torch.zeros(6, 1, V, device=DEV)
    p[:, :, 17], p[:, :, 4000] = 0.25, 0.75
    q[:, :, 17] = 1.0
    x = torch.full((6, 1), 17, dtype=torch.int64, device=DEV)
    u = torch.tensor([0.9, 0.9, 0.1, 0.1, 0.25, 0.0], device=DEV)[:, None]
    ul = torch.tensor([0.0, 1 - 2.0 ** -24, 0.0, 1 - 2.0 ** -24, 0.5, 0.3], device=DEV)
    acc, tok = _check(p, q, x, u, ul)
    assert acc.tolist() == [0, 0, 1, 1, 0, 1]           # u*q < p is strict: 0.25 is not below 0.25
    assert tok[:, 0].tolist() == [4000, 4000, 17, 17, 4000, 17]
    assert tok[2, 1] == 17 and tok[3, 1] == 4000
    # the difference is empty (q covers p) although the draft was rejected: the target itself
    q2 = torch.ones_like(q)
    acc, tok = _check(p, q2, x, torch.full_like(u, 0.5), ul)
    assert acc.tolist() == [0] * 6
    # a target without any probability, negative and NaN entries
    bad = torch.zeros(2, 2, V, device=DEV)
    bad[1, :, 3], bad[1, :, 5], bad[1, :, 9] = float("nan"), -1.0, 0.5
    acc, tok = _check(bad, q[:2], x[:2], u[:2], ul[:2])
    assert tok[0].tolist() == [-1, -1] and tok[1, 0] == 9
    # probability 0 is never accepted, even with u = 0
    p0 = p.clone()
    p0[:, :, 17] = 0
    acc, _ = _check(p0, q, x, torch.zeros_like(u), ul)
    assert acc.tolist() == [0] * 6


def test_strides_offsets_and_bad_tokens():
    p, q, x, u, ul, n = _case(4, 3, 777, torch.bfloat16, True, 9)
    big = torch.zeros(4, 4, 779, dtype=p.dtype, device=DEV)
    big[..., 1:778] = p
    bq = torch.zeros(4, 3, 780, dtype=p.dtype, device=DEV)
    bq[..., 3:] = q
    import akv
    ref = akv.verify_draft(p, q, x, u, ul, n_draft=n)
    got = akv.verify_draft(big[..., 1:778], bq[..., 3:], x.t().contiguous().t(), u, ul, n_draft=n)
    assert torch.equal(ref[0], got[0]) and torch.equal(ref[1], got[1])
    last = akv.verify_draft(p.transpose(1, 2).contiguous().transpose(1, 2), q, x, u, ul, n_draft=n)
    assert torch.equal(ref[1], last[1])
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    x2 = x.clone()
    x2[0, 0], x2[1, 0] = 777, -5
    acc, _ = _check(p, q, x2, u, ul, status=st)
    assert acc[:2].tolist() == [0, 0] and int(st) == -1


def test_distribution_is_the_targets():
    """The first token over many sequences is distributed as the target: chi-square of 8 tokens, 7 degrees of
    freedom, below 29.9 (the 1e-4 tail; the seed is fixed)."""
    import akv
    N, V = 20000, 8
    g = torch.Generator(device=DEV).manual_seed(3)
    p1 = torch.softmax(torch.randn(V, generator=g, device=DEV), -1)
    q1 = torch.softmax(torch.randn(V, generator=g, device=DEV), -1)
    x = torch.multinomial(q1.expand(N, V), 1, generator=g)
    _, tok = akv.verify_draft(p1.expand(N, 2, V).contiguous(), q1.expand(N, 1, V).contiguous(), x,
                              torch.rand(N, 1, generator=g, device=DEV), torch.rand(N, generator=g, device=DEV))
    seen = torch.bincount(tok[:, 0], minlength=V).double()
    want = p1.double() * N
    assert float(((seen - want) ** 2 / want).sum()) < 29.9


def test_refusals():
    import akv
    p, q, x, u, ul, n = _case(2, 3, 50, torch.float32, True, 1)
    ok = dict(target_probs=p, draft_probs=q, draft_tokens=x, accept_u=u, sample_u=ul, n_draft=n)
    for bad, err in ((dict(draft_probs=q.half()), ValueError), (dict(draft_probs=q[:, :2]), ValueError),
                     (dict(draft_tokens=x.int()), ValueError), (dict(draft_tokens=x[:, :2]), ValueError),
                     (dict(accept_u=u.double()), ValueError), (dict(sample_u=ul[:1]), ValueError),
                     (dict(n_draft=n.long()), ValueError), (dict(target_probs=p.double()), TypeError),
                     (dict(target_probs=p.cpu()), RuntimeError), (dict(target_probs=p[0]), ValueError)):
        with pytest.raises(err):
            akv.verify_draft(**{**ok, **bad})
    a, t = akv.verify_draft(p[:0], q[:0], x[:0], u[:0], ul[:0])
    assert a.shape == (0,) and t.shape == (0, 4)
