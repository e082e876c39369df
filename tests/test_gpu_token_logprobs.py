"""GPU: log probabilities, entropy, rank and top alternatives against their definition in 64 bits.

Tolerances, derived before the first run.  A thread adds at most V / 256 + 32 terms one by one, each sum off by
2^-24 of itself; a term e^u is off by the exponential's 2^-22, by u's two roundings (2^-23 |u|, and terms with |u| over
25 weigh nothing) and by the rescalings of a moving maximum (under 100 of 2^-22 together in the worst order):
Z off by (V / 256 + 32 + 4 + 25 * 2 + 400) 2^-24 of itself at most.  The log probability adds the roundings of its two
subtractions, 2^-23 of its size and of |x|.  The entropy is ln Z - sum(e^u u) / Z with |u| up to ln V + 25 where it
counts: the same relative error of either sum, times that.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _logits(n, v, seed, dtype, scale=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(n, v, generator=g, device=DEV) * scale).to(dtype)


def _tokens(n, v, seed):
    return torch.randint(0, v, (n,), generator=torch.Generator(device=DEV).manual_seed(seed + 1), device=DEV)


def _check(x, tokens, r, top):
    """r against 64 bits; x (n, V) finite or -inf with at least one finite logit a row."""
    n, v = x.shape
    d = x.double()
    lp = torch.log_softmax(d, -1)
    ent = -(torch.where(lp == -float("inf"), 0.0, lp) * lp.exp()).sum(-1)
    rel = (v / 256 + 32 + 4 + 50 + 400) * 2.0 ** -24
    mine = lp.gather(1, tokens[:, None])[:, 0]
    size = d.nan_to_num(neginf=0.0).abs().amax(1)
    tol = rel + 2.0 ** -23 * (size + mine.nan_to_num(neginf=0.0).abs())
    fin = mine > -float("inf")
    assert ((r.logprob.double() - mine)[fin].abs() <= tol[fin]).all()
    assert (r.logprob[~fin] == -float("inf")).all()
    import math
    assert ((r.entropy.double() - ent).abs() <= 2 * rel * (math.log(v) + 26) + 2.0 ** -22 * size).all()
    assert torch.equal(r.rank.long(), (d > d.gather(1, tokens[:, None])).sum(1) + 1)
    ids = torch.sort(d, dim=1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(r.top_tokens, ids)
    want = lp.gather(1, ids)
    fin = want > -float("inf")
    tol = (rel + 2.0 ** -23 * size)[:, None] + 2.0 ** -23 * want.nan_to_num(neginf=0.0).abs()
    assert ((r.top_logprobs.double() - want)[fin].abs() <= tol[fin]).all()
    assert (r.top_logprobs[~fin] == -float("inf")).all()


@pytest.mark.parametrize("n,v,top", [(1, 1, 1), (1, 2, 0), (3, 7, 7), (2, 31, 20), (5, 33, 32), (1, 1000, 5),
                                     (7, 8191, 1), (64, 32003, 20), (1, 151936, 32), (33, 151937, 3),
                                     (300, 5003, 8), (700, 20001, 0), (2000, 1001, 2)])
@pytest.mark.parametrize("dtype", TYPES)
def test_against_64_bits(n, v, top, dtype):
    import akv
    x, tok = _logits(n, v, n + v, dtype), _tokens(n, v, n)
    _check(x, tok, akv.token_logprobs(x, tok, top=top), top)


@pytest.mark.parametrize("dtype", TYPES)
def test_ties_order_and_extremes(dtype):
    import akv
    v = 4097
    lo = torch.finfo(dtype).min
    rows = [torch.zeros(v), torch.arange(v) % 3 * 1.0, -(torch.arange(v) % 3 * 1.0),
            torch.arange(v, dtype=torch.float32) / 64, -torch.arange(v, dtype=torch.float32) / 64,
            torch.full((v,), lo), torch.full((v,), -0.0)]
    one = torch.full((v,), -float("inf"))
    one[4000] = 2.0
    few = torch.full((v,), -float("inf"))
    few[[5, 77, 4096]] = torch.tensor([1.0, 3.0, 1.0])
    masked = torch.randn(v, generator=torch.Generator().manual_seed(3))
    masked[100:4000] = lo
    both = masked.clone()
    both[::2] = -float("inf")
    signs = torch.where(torch.arange(v) % 2 == 0, 0.0, -0.0)
    wide = torch.linspace(-3e4, 3e4, v)
    x = torch.stack(rows + [one, few, masked, both, signs, wide]).to(dtype).to(DEV)
    tok = torch.full((len(x),), 77, device=DEV)
    _check(x, tok, akv.token_logprobs(x, tok, top=9), 9)
    r = akv.token_logprobs(x, torch.full((len(x),), 4000, device=DEV), top=0)
    assert r.top_tokens.shape == (len(x), 0) and abs(float(r.logprob[7])) == 0 and float(r.entropy[7]) == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_without_a_distribution(dtype):
    import akv
    x = _logits(6, 5000, 4, dtype)
    x[0, 17] = float("nan")
    x[1, 4999] = float("inf")
    x[2] = -float("inf")
    x[3, 0] = x[3, 4998] = float("nan")
    tok = torch.tensor([1, 2, 3, 4, -1, 5000], device=DEV)
    r = akv.token_logprobs(x, tok, top=4)
    assert r.logprob.isnan().all() and (r.rank == 0).all()
    assert r.entropy[:4].isnan().all() and r.top_logprobs[:4].isnan().all() and (r.top_tokens[:4] == -1).all()
    one = akv.token_logprobs(x[4:], torch.zeros(2, dtype=torch.int64, device=DEV), top=4)
    _check(x[4:], torch.zeros(2, dtype=torch.int64, device=DEV), one, 4)
    for k in ("entropy", "top_tokens", "top_logprobs"):  # a token outside the vocabulary changes nothing else
        assert torch.equal(getattr(r, k)[4:], getattr(one, k))


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_shapes_and_alignment(dtype):
    import akv
    big = _logits(12, 2111, 9, dtype)
    for off in range(4):                                # rows from any element on, any row stride
        x = big[:, off:off + 2001 + off]
        tok = _tokens(12, 2001, off)
        _check(x, tok, akv.token_logprobs(x, tok, top=3), 3)
    y = big[:, :2000].view(3, 4, -1)[:, ::2]             # (3, 2, V)
    tok = _tokens(6, 2000, 1).view(3, 2)
    r = akv.token_logprobs(y, tok, top=2)
    assert r.logprob.shape == (3, 2) and r.top_tokens.shape == (3, 2, 2)
    flat = akv.token_logprobs(y.reshape(6, -1), tok.view(-1), top=2)
    assert all(torch.equal(a.flatten(), b.flatten()) for a, b in zip(r, flat))
    t = big.t().contiguous().t()                         # the vocabulary strided
    tok = _tokens(12, 2111, 2)
    assert all(torch.equal(a, b) for a, b in zip(akv.token_logprobs(t, tok, 2), akv.token_logprobs(big, tok, 2)))
    e = big[0].expand(5, -1)                             # one row, broadcast
    _check(e, tok[:5], akv.token_logprobs(e, tok[:5], 1), 1)
    none = akv.token_logprobs(big[:0], tok[:0], top=3)
    assert none.logprob.shape == (0,) and none.top_logprobs.shape == (0, 3)
    one = akv.token_logprobs(big[0], tok[0], top=3)      # a single row and token
    assert one.logprob.shape == () and one.top_tokens.shape == (3,)


def test_rows_past_32_bits():
    import akv
    big = torch.empty((1 << 31) + 8192, dtype=torch.float16, device=DEV)
    x = big.as_strided((3, 1003), (1 << 30, 1))
    x.copy_(_logits(3, 1003, 5, torch.float16))
    tok = _tokens(3, 1003, 6)
    _check(x, tok, akv.token_logprobs(x, tok, top=5), 5)


def test_repeated_calls_streams_and_graph():
    import akv
    x, tok = _logits(40, 30001, 7, torch.bfloat16), _tokens(40, 30001, 8)
    want = akv.token_logprobs(x, tok, top=11)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = akv.token_logprobs(x, tok, top=11)
    again = akv.token_logprobs(x, tok, top=11)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        rec = akv.token_logprobs(x, tok, top=11)
    graph.replay()
    torch.cuda.synchronize()
    for r in (other, again, rec):
        assert all(torch.equal(a, b) for a, b in zip(want, r))
    x.copy_(_logits(40, 30001, 70, torch.bfloat16))
    graph.replay()
    torch.cuda.synchronize()
    _check(x, tok, rec, 11)


def test_refusals():
    import akv
    x, tok = _logits(4, 100, 1, torch.float16), _tokens(4, 100, 1)
    for bad, err in (((x.double(), tok), TypeError), ((x.cpu(), tok.cpu()), RuntimeError), ((x, tok[:3]), ValueError),
                     ((x, tok.int()), ValueError), ((x, tok.cpu()), ValueError), ((x[:, :0], tok), ValueError)):
        with pytest.raises(err):
            akv.token_logprobs(*bad)
    for top in (-1, 33, 101):
        with pytest.raises(ValueError):
            akv.token_logprobs(x, tok, top=top)
    with pytest.raises(ValueError):
        akv.token_logprobs(x[:, :10], tok, top=11)


@pytest.mark.parametrize("v", [8192, 8200, 16384, 24581, 32767, 4099])
@pytest.mark.parametrize("dtype", TYPES)
def test_around_the_rings_batches(v, dtype):
    """Rows of whole and ragged batches, one CTA a row and several; logits of -inf in the middle and at the ends."""
    import akv
    for n in (600, 3):
        x, tok = _logits(n, v, v, dtype), _tokens(n, v, n)
        x[:, v // 2:v // 2 + 40] = -float("inf")
        x[0, :17] = x[1, -17:] = -float("inf")
        _check(x, tok, akv.token_logprobs(x, tok, top=6), 6)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logits_further_apart_than_the_type_reaches(dtype):
    """u overflows to -inf for all but the largest logit: weight 0, not NaN."""
    import akv
    x = torch.full((2, 9000), -3e38, device=DEV).to(dtype)
    x[0, 8999] = x[1, 4] = 3e38
    tok = torch.tensor([8999, 4], device=DEV)
    r = akv.token_logprobs(x, tok, top=2)
    assert (r.logprob == 0).all() and (r.entropy == 0).all() and (r.rank == 1).all()
    assert r.top_tokens.tolist() == [[8999, 0], [4, 0]]
