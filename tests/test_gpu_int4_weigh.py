"""GPU: the attention weight that cached tokens receive, against its definition in 64 bits.

Tolerance, derived before the first run.  A weight is e^(x - lse) with x = scale * (sum of s (q . (c - 8)) + (z + 8 s)
sum(q)) over the groups.  x is off by at most 2^-20 of B = scale * sum |q| (s |c - 8| + |z + 8 s|) (products of fp16
values are exact; tensor core sums of D terms keep 2^-22 of the largest partial sum, the fp32 steps after them 2^-23
each), by 2^-22 of B for the query's rounding (2^-24 of its largest element), and x - lse by 2^-22 (|x| + |lse|); the
exponential adds 2^-21.  A token's sum adds at most n terms one by one: 2^-24 n of it, n under 128 between joins, and
the joins.  Absolute floor 1e-30 for weights that underflow."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _cache(layers=1, pages=96, heads=2, dim=128, group=None, seqs=8, blocks=24):
    import akv
    return akv.Int4PagedCache(layers, pages, heads, dim, group_size=group, max_seqs=seqs, max_blocks=blocks, device=DEV,
                              track_weights=True)


def _fill(c, lens, seed=0, dtype=torch.float16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rows = torch.arange(len(lens), dtype=torch.int32, device=DEV)
    granted = c.reserve(rows, torch.tensor(lens, dtype=torch.int32, device=DEV))
    for layer in range(c.n_layers):
        k = torch.randn(len(lens), c.H, max(max(lens), 1), c.D, generator=g, device=DEV)
        k[..., 3] *= 6
        v = torch.randn(k.shape, generator=g, device=DEV)
        c.append(layer, k.to(dtype), v.to(dtype), rows, granted)
    c.check()


def _query(shape, seed, dtype, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _parts(c, layer, seq):
    """s (c - 8) and z + 8 s of K of row seq, (H, len, D) in 64 bits, from the stored bytes."""
    n, L = int(c.lens[seq]), c.layout
    nb = -(-n // 32)
    rec = c.buf[layer, c.table[seq, :nb].long()]
    code = rec[..., :16 * c.D].reshape(nb, c.H, 32, c.D // 2)
    code = torch.stack([code >> 4, code & 15], -1).flatten(-2).double() - 8
    G = c.D // c.group
    sz = rec[..., L.kp:L.kp + 128 * G].contiguous().view(torch.float16).double().view(nb, c.H, 32, G, 2)
    s, z = sz[..., 0].repeat_interleave(c.group, -1), sz[..., 1].repeat_interleave(c.group, -1)
    a, b = s * code, z + 8 * s
    return [x.transpose(0, 1).reshape(c.H, nb * 32, c.D)[:, :n] for x in (a, b)]


def _expected(c, layer, q, lse, rows, new, scale=None):
    """{seq: (sum, tolerance)} of the weights that each row's tokens get."""
    R, Hq, M, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    got = {}
    for i in range(R):
        seq, m = rows[i], new[i]
        n = int(c.lens[seq])
        w, tol = torch.zeros(n, dtype=torch.float64, device=DEV), torch.zeros(n, dtype=torch.float64, device=DEV)
        if n and m:
            a, b = _parts(c, layer, seq)
            rep = Hq // c.H
            for h in range(Hq):
                qd, l = q[i, h, :m].double(), lse[i, h, :m].double()
                ok = torch.isfinite(qd).all(-1) & torch.isfinite(l)
                qd, l = torch.where(ok[:, None], qd, 0.0), torch.where(ok, l, 0.0)
                x = qd @ (a + b)[h // rep].T * scale
                bound = qd.abs() @ (a.abs() + b.abs())[h // rep].T * abs(scale) + \
                    qd.abs().amax(-1, keepdim=True) * (a + b)[h // rep].abs().sum(-1)[None] * abs(scale) / 4
                see = (torch.arange(n, device=DEV)[None] <= (n - m + torch.arange(m, device=DEV))[:, None]) & ok[:, None]
                e = torch.where(see, (x - l[:, None]).exp(), 0.0)
                w += e.sum(0)
                tol += (e * (2.0 ** -20 * bound + 2.0 ** -22 * (x.abs() + l[:, None].abs()) + 2.0 ** -21)).sum(0)
        got[seq] = (w, tol + 2.0 ** -24 * 200 * w + 1e-30)
    return got


def _check(c, before, expected, layer=0):
    after = c.weights.double()
    for seq in range(c.max_seqs):
        n = int(c.lens[seq])
        w0 = before[layer, seq].double()
        if seq not in expected:
            assert torch.equal(after[layer, seq], w0)
            continue
        w, tol = expected[seq]
        assert torch.equal(after[layer, seq, n:], w0[n:])
        diff = (after[layer, seq, :n] - w0[:n] - w).abs()
        assert (diff <= tol + 2.0 ** -22 * (w0[:n].abs() + w)).all(), float((diff / tol).max())


LENS = [1, 2, 31, 33, 100, 319, 0, 64]


@pytest.mark.parametrize("dim,group", [(64, 64), (64, 32), (64, 16), (128, 128), (128, 64), (128, 32), (256, 256),
                                       (256, 128), (256, 64)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,rep", [(1, 1), (1, 4), (1, 7), (3, 5), (40, 3)])
def test_against_64_bits(dim, group, dtype, M, rep):
    c = _cache(heads=3, dim=dim, group=group)
    _fill(c, LENS, seed=dim + group)
    rows = [5, 0, 3, 6, 1, 4, 2]
    new = [min(M, LENS[r], m) for r, m in zip(rows, (M, M, 2, M, 1, max(1, M - 1), 0))]
    q = _query((7, 3 * rep, M, dim), 1, dtype)
    r, n = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (rows, new))
    _, lse = c.attend(0, q, r, n, return_lse=True)
    c.weights.uniform_()
    before = c.weights.clone()
    c.weigh(0, q, lse, r, n)
    c.check()
    _check(c, before, _expected(c, 0, q, lse, rows, new))


@pytest.mark.parametrize("M,rep,dim,group", [(200, 4, 128, 128), (129, 8, 64, 16), (257, 1, 256, 64), (90, 6, 128, 32)])
def test_chunks(M, rep, dim, group):
    c = _cache(heads=2, dim=dim, group=group)
    lens = [M, M + 1, 700, 450]
    _fill(c, lens, seed=3)
    new = [M, M, M - 7, 3]
    q = _query((4, 2 * rep, M, dim), 5, torch.bfloat16)
    n = torch.tensor(new, dtype=torch.int32, device=DEV)
    _, lse = c.attend(0, q, None, n, return_lse=True)
    before = c.weights.clone()
    c.weigh(0, q, lse, None, n)
    c.check()
    want = _expected(c, 0, q, lse, [0, 1, 2, 3], new)
    _check(c, before, want)
    # each query's weights sum to 1
    for i in range(4):
        assert abs(float(c.weights[0, i].double().sum()) - new[i] * 2 * rep) <= 1e-4 * new[i] * 2 * rep


def test_many_heads_and_layers():
    c = _cache(layers=3, heads=20, dim=64, pages=64)
    _fill(c, [70, 33])
    q = _query((2, 40, 5, 64), 2, torch.float16)
    for layer in (2, 0):
        _, lse = c.attend(layer, q, return_lse=True)
        before = c.weights.clone()
        c.weigh(layer, q, lse)
        _check(c, before, _expected(c, layer, q, lse, [0, 1], [5, 5]), layer)
        other = [x for x in range(3) if x != layer]
        assert torch.equal(c.weights[other], before[other])


@pytest.mark.parametrize("M", [1, 70])
def test_queries_that_count_for_nothing(M):
    c = _cache()
    _fill(c, [200, 180])
    q = _query((2, 4, M, 128), 3, torch.float16)
    _, lse = c.attend(0, q, return_lse=True)
    q[0, 0, 0, 5], q[1, 3, M - 1, 0] = float("nan"), float("inf")
    lse[0, 1, 0], lse[0, 2, M - 1], lse[1, 0, 0] = float("nan"), -float("inf"), float("inf")
    before = c.weights.clone()
    c.weigh(0, q, lse)
    c.check()
    assert torch.isfinite(c.weights).all()
    _check(c, before, _expected(c, 0, q, lse, [0, 1], [M, M]))


@pytest.mark.parametrize("M", [1, 70])
def test_bytes_past_the_end_do_not_count(M):
    """Slots past a row's end hold anything: NaN scales there reach nothing."""
    c, d = _cache(), _cache()
    for x in (c, d):
        _fill(x, [77, 101], seed=4)
    G, L = 1, c.layout
    for seq, n in ((0, 77), (1, 101)):
        page = int(c.table[seq, n // 32])
        for s in range(n % 32, 32):
            c.buf[0, page, :, L.kp + 4 * G * s:L.kp + 4 * G * (s + 1)] = 0x7F
            c.buf[0, page, :, 64 * s:64 * (s + 1)] = 0xFF
    q = _query((2, 4, M, 128), 3, torch.bfloat16)
    _, lse = d.attend(0, q, return_lse=True)
    c.weigh(0, q, lse)
    d.weigh(0, q, lse)
    c.check()
    assert torch.equal(c.weights, d.weights)


@pytest.mark.parametrize("M", [1, 70])
def test_layouts_scale_and_repetition(M):
    c, d = _cache(), _cache()
    for x in (c, d):
        _fill(x, [150, 99, 300], seed=6)
    base = _query((3, M, 4, 130), 8, torch.float16)
    q = base[..., 1:129].transpose(1, 2)                # unaligned rows, token-major
    _, lse = c.attend(0, q.contiguous(), sm_scale=0.2, return_lse=True)
    wide = torch.stack([lse, lse], -1)[..., 0]          # strided
    c.weigh(0, q, wide, sm_scale=0.2)
    d.weigh(0, q.contiguous(), lse, sm_scale=0.2)
    c.check()
    assert torch.equal(c.weights, d.weights)            # the same bits
    t = q.transpose(2, 3).contiguous().transpose(2, 3)  # channels strided
    c.weigh(0, t, lse, sm_scale=0.2)
    d.weigh(0, q, lse, sm_scale=0.2)
    assert torch.equal(c.weights, d.weights)
    _check(c, torch.zeros_like(c.weights), {k: (2 * w, 2 * t) for k, (w, t) in
                                            _expected(c, 0, q, lse, [0, 1, 2], [M] * 3, 0.2).items()})
    for scale in (-0.1, 0.0):
        c.weights.zero_()
        _, lse = c.attend(0, q, sm_scale=scale, return_lse=True)
        c.weigh(0, q, lse, sm_scale=scale)
        _check(c, torch.zeros_like(c.weights), _expected(c, 0, q, lse, [0, 1, 2], [M] * 3, scale))


@pytest.mark.parametrize("M", [1, 70])
def test_bad_rows_and_pages(M):
    c = _cache()
    _fill(c, [150, 99, 300], seed=6)
    q = _query((3, 4, M, 128), 8, torch.float16)
    lse = torch.zeros(3, 4, M, device=DEV)
    for rows in ([1, 8, 0], [1, -1, 0], [1, 1, 0]):
        c.weights.zero_()
        c.weigh(0, q, lse, torch.tensor(rows, dtype=torch.int32, device=DEV))
        with pytest.raises(RuntimeError, match="SHAPE"):
            c.check()
        good = _expected(c, 0, q[[0, 2]], lse[[0, 2]], [1, 0], [M, M])
        _check(c, torch.zeros_like(c.weights), good)
    c.weights.zero_()
    c.table[0, 2] = 1 << 20
    c.weigh(0, q, lse)
    with pytest.raises(RuntimeError, match="SHAPE"):
        c.check()
    assert (c.weights[0, 0, 64:96] == 0).all() and (c.weights[0, 0, :64] != 0).all()
    none = torch.zeros(3, dtype=torch.int32, device=DEV)
    c.weights.zero_()
    c.weigh(0, q, lse, None, none)
    c.check()
    assert (c.weights == 0).all()


@pytest.mark.parametrize("M", [1, 70])
def test_graph_streams_and_repeats(M):
    c = _cache()
    _fill(c, [150, 99, 700], seed=6)
    q = _query((3, 4, M, 128), 8, torch.float16)
    _, lse = c.attend(0, q, return_lse=True)
    c.weigh(0, q, lse)
    want = c.weights.clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    c.weights.zero_()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.weigh(0, q, lse)
    torch.cuda.synchronize()
    assert torch.equal(c.weights, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.weigh(0, q, lse)
    for _ in range(3):
        c.weights.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(c.weights, want)


def test_pool_past_32_bits():
    import akv
    c = akv.Int4PagedCache(1, 130000, 8, 128, max_seqs=2, max_blocks=16, device=DEV, track_weights=True)
    assert c.buf.numel() > 1 << 32
    d = _cache(heads=8, seqs=2, blocks=16, pages=32)
    for x in (c, d):
        _fill(x, [300, 170], seed=9)
    for j in range(10):                                 # the pages of row 0 moved to the pool's end
        c.copy_pages([int(c.table[0, j])], [129980 + j])
        c.table[0, j] = 129980 + j
    q = _query((2, 16, 1, 128), 8, torch.float16)
    _, lse = c.attend(0, q, return_lse=True)
    for x in (c, d):
        x.weigh(0, q, lse)
        x.check()
    assert torch.equal(c.weights, d.weights)


def test_reserve_and_fork_keep_weights():
    c = _cache(layers=2)
    _fill(c, [100, 50])
    c.weights.uniform_()
    w = c.weights.clone()
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    c.fork(i(0, 1, 0), i(3, 4, 5))
    c.check()
    for kid, par, n in ((3, 0, 100), (4, 1, 50), (5, 0, 100)):
        assert torch.equal(c.weights[:, kid, :n], w[:, par, :n])
        assert torch.equal(c.weights[:, kid, n:], w[:, kid, n:])
    assert torch.equal(c.weights[:, [0, 1, 2, 6, 7]], w[:, [0, 1, 2, 6, 7]])
    w = c.weights.clone()
    c.fork(i(1, 0), i(0, 6))                            # row 0 is not empty: refused, and so named twice
    with pytest.raises(RuntimeError, match="SHAPE"):
        c.check()
    assert torch.equal(c.weights[:, 0], w[:, 0]) and int(c.lens[0]) == 100
    granted = c.reserve(i(3, 1), i(7, 40))
    assert granted.tolist() == [7, 40]
    assert (c.weights[:, 3, 100:107] == 0).all() and (c.weights[:, 1, 50:90] == 0).all()
    assert torch.equal(c.weights[:, 3, :100], w[:, 3, :100]) and torch.equal(c.weights[:, 3, 107:], w[:, 3, 107:])
    assert torch.equal(c.weights[:, 1, :50], w[:, 1, :50])
    refused = c.reserve(i(3), i(100000))                # nothing granted, nothing cleared
    assert refused.tolist() == [0]
    w = c.weights.clone()
    c.status.zero_()
    c.truncate(i(3), i(20))
    assert torch.equal(c.weights, w)
    c.reserve(None, 0)
    assert torch.equal(c.weights, w)


def test_refusals():
    import akv
    c = _cache()
    _fill(c, [40, 40])
    q, lse = _query((2, 4, 3, 128), 1, torch.float16), torch.zeros(2, 4, 3, device=DEV)
    plain = akv.Int4PagedCache(1, 8, 2, 128, max_seqs=2, max_blocks=4, device=DEV)
    assert plain.weights is None
    for err, call in ((RuntimeError, lambda: plain.weigh(0, q, lse)), (ValueError, lambda: c.weigh(1, q, lse)),
                      (TypeError, lambda: c.weigh(0, q.float(), lse)), (ValueError, lambda: c.weigh(0, q[:, :3], lse)),
                      (ValueError, lambda: c.weigh(0, q, lse[:, :3])), (ValueError, lambda: c.weigh(0, q, lse.half())),
                      (RuntimeError, lambda: c.weigh(0, q.cpu(), lse)), (RuntimeError, lambda: c.weigh(0, q, lse.cpu())),
                      (ValueError, lambda: c.weigh(0, q, lse, [0, 1, 2])),
                      (ValueError, lambda: c.weigh(0, q, lse, None, [1]))):
        with pytest.raises(err):
            call()
    c.weights = c.weights[:, :1]
    with pytest.raises(ValueError):
        c.weigh(0, q, lse)
    with pytest.raises(ValueError):
        c.reserve(None, 1)


@pytest.mark.parametrize("M,group", [(2, 64), (40, 64), (40, 16)])
def test_more_rows_than_a_launch_lists(M, group):
    R = 1100
    c = _cache(pages=2 * R, heads=1, dim=64, group=group, seqs=R, blocks=2)
    lens = [M + i % 20 for i in range(R)]
    _fill(c, lens, seed=R)
    q = _query((R, 1, M, 64), 3, torch.float16)
    lse = torch.randn(R, 1, M, device=DEV) + 5
    c.weigh(0, q, lse)
    c.check()
    all_of_it = c.weights.clone()
    for i in (0, 1023, 1024, R - 1):
        w, tol = _expected(c, 0, q[i:i + 1], lse[i:i + 1], [i], [M])[i]
        assert ((all_of_it[0, i, :lens[i]].double() - w).abs() <= tol).all()
        assert (all_of_it[0, i, lens[i]:] == 0).all()


def test_nothing_to_do():
    c = _cache(pages=8, blocks=4)
    _fill(c, [40, 5], seed=1)
    for shape in ((0, 4, 5, 128), (2, 4, 0, 128)):
        c.weigh(0, _query(shape, 1, torch.float16), torch.zeros(shape[:3], device=DEV),
                torch.arange(shape[0], dtype=torch.int32, device=DEV))
    c.check()
    assert not c.weights.any()


@pytest.mark.parametrize("group", [128, 64, 32])
@pytest.mark.parametrize("columns", [15, 16, 17, 31, 32, 33, 48])
def test_both_kernels_at_their_boundary(group, columns):
    c = _cache(heads=2, group=group)
    _fill(c, [200, 33, 64], seed=columns)
    q = _query((3, 2, columns, 128), 4, torch.bfloat16)
    new = [columns, min(33, columns), columns]
    n = torch.tensor(new, dtype=torch.int32, device=DEV)
    rows = torch.arange(3, dtype=torch.int32, device=DEV)
    lse = torch.randn(3, 2, columns, device=DEV) + 6
    before = c.weights.clone()
    c.weigh(0, q, lse, rows, n)
    c.check()
    _check(c, before, _expected(c, 0, q, lse, [0, 1, 2], new))
