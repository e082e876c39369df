"""GPU: attention weight with many rows named: each once, in any order, at the price of unnamed ones."""
import pytest
import torch

from test_gpu_int4_weigh import DEV, _cache, _fill, _query

pytestmark = pytest.mark.gpu

# the two kernels: 2 and 40 query columns
COLUMNS = [(2, 64), (40, 64), (40, 16)]


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _close(a, b):
    """Sums of up to 40 positive terms in another order, each partial sum rounded: 2 * 41 * 2^-24 of them."""
    return bool(((a - b).abs() <= 82 * 2.0 ** -24 * b.abs()).all())


@pytest.mark.parametrize("M,group", COLUMNS)
@pytest.mark.parametrize("seqs", [1100, 70000])
def test_named_rows_count_once(M, group, seqs):
    """1,100 of the cache's rows in another order, two launches; some of them twice, the second time near and far."""
    R, step = 1100, seqs // 1100
    c = _cache(pages=2 * R, heads=1, dim=64, group=group, seqs=seqs, blocks=2)
    order = torch.randperm(R, generator=torch.Generator().manual_seed(3))
    rows = _ints((order * step).tolist())
    lens = _ints([M + i % 20 for i in range(R)])
    granted = c.reserve(rows, lens)
    k = torch.randn(R, 1, M + 20, 64, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).half()
    c.append(0, k, k, rows, granted)
    q = _query((R, 1, M, 64), 3, torch.float16)
    lse = torch.randn(R, 1, M, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV) + 5
    want = torch.zeros_like(c.weights)
    for a in range(0, R, 10):                                # few at a time
        c.weights.zero_()
        c.weigh(0, q[a:a + 10], lse[a:a + 10], rows[a:a + 10])
        want += c.weights
    c.weights.zero_()
    c.weigh(0, q, lse, rows)
    c.check()
    assert _close(c.weights, want)
    # repeats: of the one before, of the first, across the launches, of two others alike
    twice = rows.clone()
    for i, j in ((1, 0), (500, 499), (1022, 0), (1024, 1023), (1099, 3), (700, 3), (1098, 1030)):
        twice[i] = rows[j]
        want[0, rows[i]] = 0
    c.weights.zero_()
    c.weigh(0, q, lse, twice)
    with pytest.raises(RuntimeError, match="SHAPE"):
        c.check()
    assert _close(c.weights, want)


def test_rows_a_power_of_two_apart():
    c = _cache(pages=64, heads=1, dim=64, group=64, seqs=131073, blocks=1)
    rows = _ints([32768 * k for k in (4, 0, 1, 2, 3)] + [5, 32773, 5])
    granted = c.reserve(rows[:7], 20)
    k = torch.randn(7, 1, 20, 64, device=DEV).half()
    c.append(0, k, k, rows[:7], granted)
    for M in (2, 40):
        q, lse = _query((8, 1, M, 64), 3, torch.float16), torch.zeros(8, 1, M, device=DEV)
        c.weights.zero_()
        c.weigh(0, q[:7], lse[:7], rows[:7])
        c.check()
        want = c.weights.clone()
        assert (want[0, rows[:7].long(), :20] > 0).all()
        c.weights.zero_()
        c.weigh(0, q, lse, rows)
        with pytest.raises(RuntimeError, match="SHAPE"):
            c.check()
        assert _close(c.weights, want)


@pytest.mark.parametrize("M,group", COLUMNS)
def test_names_cost_little(M, group):
    """1,024 rows of 300 tokens: naming them, which a serving loop does, takes no more than half as long again."""
    R = 1024
    c = _cache(pages=10 * R, heads=2, dim=64, group=group, seqs=R, blocks=10)
    _fill(c, [300] * R)
    q = _query((R, 2, M, 64), 3, torch.float16)
    lse = torch.zeros(R, 2, M, device=DEV) + 6

    def us(rows):
        best = 1e9
        for _ in range(30):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            torch.cuda.synchronize()
            start.record()
            for _ in range(5):
                c.weigh(0, q, lse, rows)
            end.record()
            torch.cuda.synchronize()
            best = min(best, start.elapsed_time(end) * 200)
        return best

    rows = torch.arange(R, dtype=torch.int32, device=DEV)
    us(rows)
    plain, named = us(None), us(rows)
    print(f"{M} columns, groups of {group}: {plain:.1f} us, named {named:.1f}")
    assert named <= 1.5 * plain
