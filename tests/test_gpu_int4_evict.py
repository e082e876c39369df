"""GPU: eviction from the 4-bit paged cache against a plain restatement, byte for byte.

Everything here is whole numbers or copies: the score of a token is the fp64 sum of its weights rounded once to fp32,
so it is the same in any order of the layers (fp64 sums of a few fp32 numbers differ by 2^-52), and ties go to the
earliest token.  Nothing is compared with a tolerance except the attention over what stays."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _cache(layers=3, pages=200, heads=2, dim=64, group=None, seqs=8, blocks=20):
    import akv
    return akv.Int4PagedCache(layers, pages, heads, dim, group_size=group, max_seqs=seqs, max_blocks=blocks, device=DEV,
                              track_weights=True)


def _i(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _fill(c, lens, seed=0):
    """Rows of these lengths, every byte of the pool random."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    c.buf.copy_(torch.randint(0, 256, c.buf.shape, generator=g, device=DEV, dtype=torch.uint8))
    rows = torch.arange(len(lens), dtype=torch.int32, device=DEV)
    c.reserve(rows, torch.tensor(lens, dtype=torch.int32, device=DEV))
    c.weights.copy_((torch.randn(c.weights.shape, generator=g, device=DEV) * 2).exp())
    c.check()


def _tokens(c, buf, table, seq, n):
    """The bytes of row seq's tokens in every layer and head, [layer, head, token, byte]."""
    L, G = c.layout, c.D // c.group
    buf, table = buf.cpu().numpy(), table.cpu().numpy()
    out = np.zeros((c.n_layers, c.H, n, c.D + 8 * G), np.uint8)
    for t in range(n):
        rec, s = buf[:, table[seq, t // 32]], t % 32
        out[:, :, t] = np.concatenate([rec[:, :, L.kc + s * c.D // 2:L.kc + (s + 1) * c.D // 2],
                                       rec[:, :, L.vc + s * c.D // 2:L.vc + (s + 1) * c.D // 2],
                                       rec[:, :, L.kp + s * 4 * G:L.kp + (s + 1) * 4 * G],
                                       rec[:, :, L.vp + s * 4 * G:L.vp + (s + 1) * 4 * G]], -1)
    return out


def _kept(c, w, seq, n, keep, first, recent):
    if n <= keep:
        return list(range(n))
    s = w[:, seq, :n].double().sum(0).float().cpu().numpy()
    s = np.where(np.isnan(s), -np.inf, s)
    nan = np.isnan(w[:, seq, :n].double().sum(0).float().cpu().numpy())
    forced = [t for t in range(n) if t < first or t >= n - recent]
    rest = sorted((t for t in range(n) if first <= t < n - recent), key=lambda t: (nan[t], -s[t], t))
    return sorted(forced + rest[:keep - len(forced)])


def _run(c, rows, keep, first=0, recent=0, refused=()):
    """One eviction, checked: tokens, weights, kept, lengths, reference counts, free pages, untouched rows."""
    buf, table, lens, w = c.buf.clone(), c.table.clone(), c.lens.tolist(), c.weights.clone()
    which = list(range(c.max_seqs)) if rows is None else list(rows)
    kept = c.evict(None if rows is None else _i(*rows), keep, first, recent)
    assert kept.shape == (len(which), keep) and kept.dtype is torch.int32
    done = set()
    for i, seq in enumerate(which):
        got = [t for t in kept[i].tolist() if t >= 0]
        assert kept[i].tolist() == got + [-1] * (keep - len(got))
        if seq in done or seq in refused or not 0 <= seq < c.max_seqs:
            assert got == []
            continue
        done.add(seq)
        want = _kept(c, w, seq, lens[seq], keep, first, recent)
        assert got == want and int(c.lens[seq]) == len(want)
        np.testing.assert_array_equal(_tokens(c, c.buf, c.table, seq, len(want)),
                                      _tokens(c, buf, table, seq, lens[seq])[:, :, want])
        assert torch.equal(c.weights[:, seq, :len(want)].contiguous().view(torch.int32),
                           w[:, seq][:, want].contiguous().view(torch.int32))   # the bits: NaN among them
        nb = -(-len(want) // 32)
        if lens[seq] > keep:
            assert (c.table[seq, nb:] == -1).all()
    for seq in range(c.max_seqs):
        if seq not in done:                              # others keep their pages and what is on them
            assert int(c.lens[seq]) == lens[seq] and torch.equal(c.table[seq], table[seq])
            assert torch.equal(c.weights[:, seq], w[:, seq])
            np.testing.assert_array_equal(_tokens(c, c.buf, c.table, seq, lens[seq]),
                                          _tokens(c, buf, table, seq, lens[seq]))
    refs = torch.zeros_like(c.refs)
    for seq in range(c.max_seqs):
        nb = -(-int(c.lens[seq]) // 32)
        refs.index_add_(0, c.table[seq, :nb].long(), torch.ones(nb, dtype=torch.int32, device=DEV))
    assert torch.equal(refs, c.refs)
    bits = c.free_bits.cpu().numpy().view(np.uint32)
    free = [p for p in range(c.n_pages) if bits[p // 32] >> (p % 32) & 1]
    assert free == [p for p in range(c.n_pages) if int(refs[p]) == 0]
    return kept


@pytest.mark.parametrize("dim,group", [(64, 64), (64, 32), (64, 16), (128, 128), (128, 64), (128, 32), (256, 256),
                                       (256, 128), (256, 64)])
def test_shapes(dim, group):
    c = _cache(dim=dim, group=group, heads=3)
    _fill(c, [500, 33, 640, 129, 1, 0, 128, 300], seed=dim + group)
    _run(c, None, 128, first=4, recent=30)
    c.check()


@pytest.mark.parametrize("keep,first,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (31, 0, 0), (32, 3, 3), (33, 0, 33),
                                               (64, 64, 0), (200, 1, 150), (499, 0, 0), (500, 0, 0), (600, 100, 100),
                                               (5000, 2500, 2500)])
def test_budgets(keep, first, recent):
    c = _cache(layers=2, blocks=30, seqs=5)
    _fill(c, [500, 900, 501, 31, 0], seed=keep)
    _run(c, None, keep, first, recent)
    c.check()


def test_ties_and_odd_weights():
    c = _cache(layers=2)
    _fill(c, [400, 400, 400, 400, 400, 400])
    w = c.weights
    w[:, 0] = 0.0                                        # all equal: the earliest stay
    w[:, 1] = -0.0
    w[:, 1, ::3] = 0.0
    w[:, 2] = (torch.arange(w.shape[2], device=DEV) % 4).float()
    w[:, 3] = -w[:, 3]                                   # negative weights order like any
    w[0, 4, ::2] = float("nan")                          # NaN below all
    w[:, 5, 10:300] = float("inf")
    w[0, 5, 100] = -float("inf")                         # inf - inf: NaN
    _run(c, [3, 0, 5, 1, 4, 2], 150, 0, 5)
    c.check()


def test_weights_far_apart_between_layers():
    c = _cache(layers=20, pages=60, heads=1)
    _fill(c, [600])
    g = torch.Generator(device=DEV).manual_seed(1)
    c.weights.copy_(torch.rand(c.weights.shape, generator=g, device=DEV) *
                    10.0 ** torch.randint(-12, 12, c.weights.shape, generator=g, device=DEV))
    _run(c, [0], 333)
    c.check()


def test_only_the_last_tokens_go():
    """Nothing moves: shared pages stay shared."""
    c = _cache()
    _fill(c, [300, 70])
    c.fork(_i(0, 1), _i(3, 4))
    c.weights[:, 3] = -torch.arange(640, device=DEV).float()
    table = c.table.clone()
    _run(c, [3], 130)
    c.check()
    assert torch.equal(c.table[3, :5], table[0, :5])


def test_shared_pages():
    c = _cache(pages=120)
    _fill(c, [450, 200, 90])
    c.fork(_i(0, 0, 1), _i(4, 5, 6))
    c.weights[:, 0, :100] += 1e6                         # the first pages of row 0 and its forks stay shared
    c.weights[:, 4:6, :100] += 1e6
    kept = _run(c, [4, 0, 6, 1], 160, 0, 20)
    assert kept[0, 99] == 99
    assert torch.equal(c.table[4, :3], c.table[5, :3]) and int(c.refs[c.table[5, 0].long()]) == 3
    c.check()
    _run(c, None, 64, 2, 2)
    c.check()
    c.free(None)
    assert c.free_pages() == 120


def test_partial_page_shared_after_the_end():
    """A fork of a partly filled page, appended to after the eviction: copy on write still holds."""
    c = _cache(layers=1)
    _fill(c, [200])
    c.fork(_i(0), _i(1))
    _run(c, [1], 50, 10, 10)
    c.fork(_i(1), _i(2))
    g = c.reserve(_i(1, 2), 3)
    assert g.tolist() == [3, 3]
    k = torch.randn(2, 2, 3, 64, device=DEV).half()
    before = _tokens(c, c.buf, c.table, 1, 50)
    c.append(0, k, k, _i(1, 2), g)
    c.check()
    for seq in (1, 2):
        np.testing.assert_array_equal(_tokens(c, c.buf, c.table, seq, 50), before)


def test_pool_runs_out():
    c = _cache(pages=16 + 7 + 2, seqs=6)
    _fill(c, [512, 200])                                 # 16 and 7 pages: two free ones
    c.fork(_i(0, 1, 1), _i(2, 3, 4))
    c.weights[:, 2, 60:70] = -1.0                        # row 2 writes pages 1 and 2 (of 64 tokens kept: page 1)
    c.weights[:, 2, :60] = 9e9
    _run(c, [2, 3, 4, 0], 64, 0, 1, refused=(3, 4, 0))
    with pytest.raises(RuntimeError, match="EXHAUSTED"):
        c.check()


def test_bad_and_repeated_rows():
    c = _cache()
    _fill(c, [300, 200, 100])
    _run(c, [1, 9, 1, -1, 0], 64)
    with pytest.raises(RuntimeError, match="SHAPE"):
        c.check()
    c = _cache()
    _fill(c, [300, 200, 100])
    c.lens[1] = 100000                                   # no length: refused, the others go
    kept = c.evict(None, 64)
    with pytest.raises(RuntimeError, match="SHAPE"):
        c.check()
    assert (kept[1] == -1).all() and c.lens.tolist()[:3] == [64, 100000, 64]


def test_bad_page_numbers():
    c = _cache()
    _fill(c, [300, 200])
    buf, w = c.buf.clone(), c.weights.clone()
    c.table[0, 1], c.table[0, 8] = -5, 1 << 20
    good = c.table[1].clone()
    c.evict(_i(0), 100)
    with pytest.raises(RuntimeError, match="SHAPE"):
        c.check()
    assert int(c.lens[0]) == 100 and torch.equal(c.table[1], good)
    assert torch.equal(c.buf[:, good[:7].long()], buf[:, good[:7].long()]) and torch.equal(c.weights[:, 1], w[:, 1])


def test_attention_over_what_stays():
    """An evicted row attends like one that was given the kept tokens alone."""
    import akv
    c = _cache(layers=1, dim=128, heads=2)
    d = _cache(layers=1, dim=128, heads=2)
    g = torch.Generator(device=DEV).manual_seed(2)
    k, v = (torch.randn(1, 2, 300, 128, generator=g, device=DEV).half() for _ in range(2))
    c.append(0, k, v, _i(0), c.reserve(_i(0), 300))
    q = torch.randn(1, 8, 16, 128, generator=g, device=DEV).half()
    _, lse = c.attend(0, q, _i(0), return_lse=True)
    c.weigh(0, q, lse, _i(0))
    kept = c.evict(_i(0), 77, first=2, recent=16)[0].long()
    d.append(0, k[:, :, kept], v[:, :, kept], _i(0), d.reserve(_i(0), 77))
    new = torch.randn(1, 2, 1, 128, generator=g, device=DEV).half()
    outs = []
    for x in (c, d):
        granted = x.reserve(_i(0), 1)
        x.append(0, new, new, _i(0), granted)
        outs.append(x.attend(0, q[:, :, :1], _i(0), granted))
        x.check()
    assert torch.equal(outs[0], outs[1])
    assert torch.equal(c.weights[0, 0, 77:78], torch.zeros(1, device=DEV))
    assert isinstance(c, akv.Int4PagedCache)


def test_graph_and_side_stream():
    c = _cache()
    _fill(c, [500, 300, 640])
    state, buf, w = c.page_state(), c.buf.clone(), c.weights.clone()
    want = c.evict(None, 100, 2, 10)
    after = (c.buf.clone(), c.page_state(), c.weights.clone())

    def back():
        c.set_page_state(state)
        c.buf.copy_(buf)
        c.weights.copy_(w)

    back()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kept = c.evict(None, 100, 2, 10)
    torch.cuda.synchronize()
    assert torch.equal(kept, want) and torch.equal(c.buf, after[0]) and torch.equal(c.page_state(), after[1])
    back()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = c.evict(None, 100, 2, 10)
    for _ in range(2):
        back()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kept, want) and torch.equal(c.buf, after[0])
        assert torch.equal(c.page_state(), after[1]) and torch.equal(c.weights, after[2])
    c.check()


def test_many_rows_and_long_ones():
    c = _cache(layers=1, pages=5000, heads=1, seqs=1100, blocks=4)
    _fill(c, [20 + (i * 37) % 100 for i in range(1100)])
    w, lens = c.weights.clone(), c.lens.tolist()
    kept = c.evict(None, 40, 1, 3).tolist()
    c.check()
    for seq in range(0, 1100, 7):
        assert [t for t in kept[seq] if t >= 0] == _kept(c, w, seq, lens[seq], 40, 1, 3)
    d = _cache(layers=1, pages=3200, heads=1, seqs=2, blocks=3125)
    _fill(d, [99999, 5])
    _run(d, [0], 33333, 5, 1000)
    d.check()


def test_refusals():
    import akv
    c = _cache()
    _fill(c, [100])
    plain = akv.Int4PagedCache(1, 8, 2, 128, max_seqs=2, max_blocks=4, device=DEV)
    with pytest.raises(RuntimeError):
        plain.evict(None, 4)
    for bad in ((0, 0, 0), (-1, 0, 0), (10, 11, 0), (10, 5, 6), (10, -1, 0), (10, 0, -1), (1 << 31, 0, 0)):
        with pytest.raises(ValueError):
            c.evict(None, *bad)
    for rows in (torch.zeros(2, 2, dtype=torch.int32, device=DEV), torch.zeros(2, device=DEV), _i(0).cpu()):
        with pytest.raises(ValueError):
            c.evict(rows, 10)
    assert c.evict(_i(), 10).shape == (0, 10)
    c.check()


@pytest.mark.parametrize("dim,group", [(64, 64), (64, 32), (64, 16), (128, 128), (128, 64), (128, 32), (256, 256),
                                       (256, 128), (256, 64)])
def test_many_blocks(dim, group):
    """Enough rows, layers and heads for the moves' smaller blocks, rows of several of their steps."""
    c = _cache(layers=8, pages=150, heads=4, dim=dim, group=group, blocks=20)
    _fill(c, [600, 1, 333, 640, 64, 97], seed=dim + group)
    c.fork([3], [6])
    c.check()
    _run(c, [3, 0, 4, 2, 1], 300, first=3, recent=11)


def test_no_rows():
    c = _cache()
    _fill(c, [100])
    buf, table = c.buf.clone(), c.table.clone()
    assert c.evict(torch.empty(0, dtype=torch.int32, device=DEV), 5).shape == (0, 5)
    assert torch.equal(c.buf, buf) and torch.equal(c.table, table) and c.lens.tolist()[0] == 100
    c.check()
