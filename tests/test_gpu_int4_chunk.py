"""GPU: attention of a chunk of new tokens over the 4-bit paged cache against the formula in 64 bits.

Tolerances, derived before the first run.  With weights w_t (sum 1), values V_t and out = sum w_t V_t:
  * a score off by d_t moves the output by at most sum w_t d_t |V_t - out| (and second order terms, d_t < 0.1: 10 % more);
    d_t = scale * sum |q| |K_t| * k, k = 2^-11 for a bf16 query (K rounded to fp16) or 2^-20 (two terms, fp32 sums), and
    2^-20 of the same sum for the query's scaling and the tensor cores' sums;
  * weights rounded to fp16 once (bf16): 2^-11 sum w_t |V_t|, or twice (fp16): 2^-20 of it;
  * V rounded to fp16 once: 2^-11 sum w_t |V_t|, values below fp16's normal range 2^-25 more;
  * the output's own rounding, 2^-11 or 2^-8 of it, and fp32 sums: 2^-20 of the largest |V|.
The lse is off by at most the largest d_t, and fp32's 2^-20 of its size and of the largest score + 1e-5."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _cache(layers=1, pages=200, heads=2, dim=128, group=None, seqs=8, blocks=40):
    import akv
    return akv.Int4PagedCache(layers, pages, heads, dim, group_size=group, max_seqs=seqs, max_blocks=blocks, device=DEV)


def _fill(c, lens, seed=0, dtype=torch.float16, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rows = torch.arange(len(lens), dtype=torch.int32, device=DEV)
    granted = c.reserve(rows, torch.tensor(lens, dtype=torch.int32, device=DEV))
    for layer in range(c.n_layers):
        k = torch.randn(len(lens), c.H, max(max(lens), 1), c.D, generator=g, device=DEV) * scale
        k[..., 3] *= 6
        v = torch.randn(k.shape, generator=g, device=DEV) * scale
        c.append(layer, k.to(dtype), v.to(dtype), rows, granted)
    c.check()


def _query(shape, seed, dtype, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _values(c, layer, seq):
    """K and V of row seq, (H, len, D) in 64 bits, from the stored bytes."""
    n, L = int(c.lens[seq]), c.layout
    nb = -(-n // 32)
    rec = c.buf[layer, c.table[seq, :nb].long()]
    out, G = [], c.D // c.group
    for c0, p0 in ((L.kc, L.kp), (L.vc, L.vp)):
        code = rec[..., c0:c0 + 16 * c.D].reshape(nb, c.H, 32, c.D // 2)
        code = torch.stack([code >> 4, code & 15], -1).flatten(-2).double()
        sz = rec[..., p0:p0 + 128 * G].contiguous().view(torch.float16).double().view(nb, c.H, 32, G, 2)
        x = code * sz[..., 0].repeat_interleave(c.group, -1) + sz[..., 1].repeat_interleave(c.group, -1)
        out.append(x.transpose(0, 1).reshape(c.H, nb * 32, c.D)[:, :n])
    return out


def _check(c, q, out, lse, rows, new, layer=0, scale=None):
    R, Hq, M, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    bf = q.dtype is torch.bfloat16
    rep = Hq // c.H
    worst = 0.0
    for i in range(R):
        seq, m = rows[i], new[i]
        n = int(c.lens[seq]) if 0 <= seq < c.max_seqs else 0
        m = min(m, M)
        assert (out[i, :, m:] == 0).all()
        if lse is not None:
            assert (lse[i, :, m:] == -math.inf).all()
        if not m:
            continue
        k, v = _values(c, layer, seq)
        see = torch.arange(n, device=DEV)[None] <= (n - m + torch.arange(m, device=DEV))[:, None]
        for h in range(Hq):
            qd, kd, vd = q[i, h, :m].double(), k[h // rep], v[h // rep]
            x = torch.where(see, qd @ kd.T * scale, -math.inf)
            w = torch.softmax(x, -1)
            want = w @ vd
            d = abs(scale) * (qd.abs() @ kd.abs().T) * ((2.0 ** -11 if bf else 2.0 ** -20) + 2.0 ** -20)
            d += abs(scale) * qd.abs().amax(-1, keepdim=True) * kd.abs().sum(-1)[None] * 2.0 ** -24
            wd = w * d
            moved = wd @ vd.abs() + wd.sum(-1, keepdim=True) * want.abs()      # >= sum w d |V - out|
            vabs = w @ vd.abs()
            tol = 1.1 * moved + vabs * (2 * 2.0 ** -11 if bf else 2.0 ** -11 + 2.0 ** -20) + 2.0 ** -25 + \
                (2.0 ** -8 if bf else 2.0 ** -11) * want.abs() + 2.0 ** -20 * vd.abs().max()
            diff = (out[i, h, :m].double() - want).abs()
            worst = max(worst, float((diff / tol).max()))
            assert (diff <= tol).all(), (i, h, float((diff / tol).max()))
            if lse is not None:
                want = torch.logsumexp(x, -1)
                top = x.masked_fill(~see, 0.0).abs().amax(-1)
                tol = d.amax(-1) + 2.0 ** -20 * (want.abs() + top) + 1e-5
                assert ((lse[i, h, :m].double() - want).abs() <= tol).all()
    return worst


@pytest.mark.parametrize("dim,group", [(64, 64), (64, 32), (64, 16), (128, 128), (128, 64), (128, 32), (256, 256),
                                       (256, 128), (256, 64)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_against_64_bits(dim, group, dtype):
    c = _cache(heads=2, dim=dim, group=group)
    lens = [150, 1, 640, 333, 0, 129, 128]
    _fill(c, lens, seed=dim + group)
    rows, new = [2, 0, 6, 1, 4, 3, 5], [100, 100, 99, 1, 0, 37, 2]
    q = _query((7, 6, 100, dim), 1, dtype)
    r, n = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (rows, new))
    out, lse = c.attend_chunk(0, q, r, n, return_lse=True)
    c.check()
    _check(c, q, out, lse, rows, new)


@pytest.mark.parametrize("M,rep,lens", [(1, 1, [1]), (1, 1, [1000]), (2, 8, [2, 65]), (16, 1, [1280, 16]),
                                        (127, 2, [127, 128]), (128, 1, [128, 129]), (129, 3, [129, 700]),
                                        (257, 1, [257, 300]), (300, 4, [300]), (512, 2, [1280]), (65, 16, [66, 1025])])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_chunk_sizes(M, rep, lens, dtype):
    c = _cache(heads=1)
    _fill(c, lens, seed=M)
    q = _query((len(lens), rep, M, 128), 2, dtype)
    out, lse = c.attend_chunk(0, q, return_lse=True)
    c.check()
    _check(c, q, out, lse, list(range(len(lens))), [M] * len(lens))


@pytest.mark.parametrize("dim,dtype", [(64, torch.bfloat16), (128, torch.float16), (256, torch.bfloat16)])
def test_many_units_and_parts(dim, dtype):
    """More units than CTAs, cut where the shares end; a few long rows among short ones."""
    c = _cache(heads=5, dim=dim, pages=900, seqs=24, blocks=130)
    lens = [4000 if r in (3, 17) else 100 + 31 * r for r in range(24)]
    _fill(c, lens, seed=7)
    new = [min(n, 64 + 3 * r) for r, n in enumerate(lens)]
    q = _query((24, 15, max(new), dim), 3, dtype)
    out, lse = c.attend_chunk(0, q, None, torch.tensor(new, dtype=torch.int32, device=DEV), return_lse=True)
    c.check()
    _check(c, q, out, lse, list(range(24)), new)


def test_like_attend():
    """fp16: the decode kernel's results to both kernels' roundings; layers apart."""
    c = _cache(layers=2, heads=2)
    _fill(c, [700, 90])
    q = _query((2, 8, 40, 128), 4, torch.float16)
    for layer in (1, 0):
        a, la = c.attend(layer, q, return_lse=True)
        b, lb = c.attend_chunk(layer, q, return_lse=True)
        _check(c, q, b, lb, [0, 1], [40, 40], layer)
        assert (la - lb).abs().max() <= 1e-4 and (a.float() - b.float()).abs().max() <= 2.0 ** -9 * 8


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_query_extremes(dtype):
    c = _cache()
    _fill(c, [300])
    q = _query((1, 4, 100, 128), 5, dtype)
    q[0, 0, 3, 7], q[0, 1, 50, 0], q[0, 3, 99, 127] = float("nan"), float("inf"), -float("inf")
    q[0, 2, 10] = 0
    q[0, 2, 11] *= 1e-4
    q[0, 2, 12] *= 60
    if dtype is torch.bfloat16:
        q[0, 2, 13] *= 1e-30
        q[0, 2, 14, 5] = 3e5
    out, lse = c.attend_chunk(0, q, return_lse=True)
    c.check()
    bad = ~torch.isfinite(q).all(-1)
    assert out[bad].isnan().all() and lse[bad].isnan().all()
    assert torch.isfinite(out[~bad]).all()
    fine = torch.where(bad[..., None], 0.0, q)
    clean, cl = c.attend_chunk(0, fine, return_lse=True)
    assert torch.equal(out[~bad], clean[~bad]) and torch.equal(lse[~bad], cl[~bad])
    _check(c, fine, clean, cl, [0], [100])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scale", [-0.1, 0.0, 0.5, 1e-3])
def test_scales(dtype, scale):
    c = _cache()
    _fill(c, [300, 64])
    q = _query((2, 4, 64, 128), 5, dtype)
    out, lse = c.attend_chunk(0, q, sm_scale=scale, return_lse=True)
    _check(c, q, out, lse, [0, 1], [64, 64], scale=scale)


@pytest.mark.parametrize("dim,group", [(64, 64), (128, 32), (128, 128), (256, 128)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_values_at_the_ends_of_fp16(dim, group, dtype):
    """c * s + z past 65504 by its rounding: held to it (read() does so too), never infinite; tiny values too."""
    c = _cache(heads=1, dim=dim, group=group)
    x = torch.randn(1, 1, 200, dim, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    v = x.clone()
    v[0, 0, 5:90, ::2], v[0, 0, 5:90, 1::2] = 65504.0, -65504.0
    v[0, 0, 90:120] *= 1e-6
    c.append(0, x.half(), v.half(), [0], c.reserve([0], 200))
    q = _query((1, 3, 150, dim), 6, dtype)
    out = c.attend_chunk(0, q, [0])
    c.check()
    assert torch.isfinite(out).all()
    k64, v64 = _values(c, 0, 0)
    over = v64.abs().max() - 65504.0                 # how far the formula's values pass it: clamped there
    see = torch.arange(200, device=DEV)[None] <= (50 + torch.arange(150, device=DEV))[:, None]
    for h in range(3):
        xs = torch.where(see, q[0, h].double() @ k64[0].T * dim ** -0.5, -math.inf)
        w = torch.softmax(xs, -1)
        d = dim ** -0.5 * (q[0, h].double().abs() @ k64[0].abs().T) * (2.0 ** -11 if dtype is torch.bfloat16 else 2.0 ** -20)
        want, vabs = w @ v64[0], w @ v64[0].abs()
        tol = 1.1 * (w * d) @ v64[0].abs() + 1.1 * (w * d).sum(-1, keepdim=True) * want.abs() + vabs * 2.0 ** -9 + over + \
            (2.0 ** -8 if dtype is torch.bfloat16 else 2.0 ** -11) * want.abs() + 2.0 ** -20 * 65504
        assert ((out[0, h].double() - want).abs() <= tol).all()


def test_bytes_past_the_end_do_not_count():
    c, d = _cache(), _cache()
    for x in (c, d):
        _fill(x, [77, 301], seed=4)
    c.buf[0, [p for p in range(200) if int(c.refs[p]) == 0]] = 0x7F
    L = c.layout
    for seq, n in ((0, 77), (1, 301)):
        page = int(c.table[seq, n // 32])
        for s in range(n % 32, 32):
            for p0, c0 in ((L.kp, L.kc), (L.vp, L.vc)):
                c.buf[0, page, :, p0 + 4 * s:p0 + 4 * (s + 1)] = 0x7F
                c.buf[0, page, :, c0 + 64 * s:c0 + 64 * (s + 1)] = 0xFF
    for dtype in (torch.float16, torch.bfloat16):
        q = _query((2, 4, 70, 128), 3, dtype)
        a, b = c.attend_chunk(0, q, return_lse=True), d.attend_chunk(0, q, return_lse=True)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    c.check()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_layouts(dtype):
    c = _cache()
    _fill(c, [150, 99, 300], seed=6)
    base = _query((3, 90, 4, 130), 8, dtype)
    q = base[..., 1:129].transpose(1, 2)                 # unaligned rows, token-major
    want, lse = c.attend_chunk(0, q.contiguous(), return_lse=True)
    out, l2 = c.attend_chunk(0, q, return_lse=True)
    assert torch.equal(out, want) and torch.equal(l2, lse)
    t = q.transpose(2, 3).contiguous().transpose(2, 3)   # channels strided
    assert torch.equal(c.attend_chunk(0, t), want)
    guard = torch.full((3, 4, 92, 131), 7.0, dtype=dtype, device=DEV)
    given = guard[:, :, 1:91, 2:130]                     # an unaligned output among other data
    assert c.attend_chunk(0, q, out=given) is given and torch.equal(given, want)
    guard[:, :, 1:91, 2:130] = 7.0
    assert (guard == 7.0).all()
    tm = torch.empty(3, 90, 4, 128, dtype=dtype, device=DEV).transpose(1, 2)
    assert torch.equal(c.attend_chunk(0, q, out=tm), want)
    wide = q[:, :1].expand(3, 6, 90, 128)                # one head, broadcast
    assert torch.equal(c.attend_chunk(0, wide)[:, 4], c.attend_chunk(0, wide.contiguous())[:, 4])


def test_bad_rows_and_pages():
    c = _cache()
    _fill(c, [150, 99, 300], seed=6)
    q = _query((3, 4, 70, 128), 8, torch.bfloat16)
    good = c.attend_chunk(0, q)
    out, lse = c.attend_chunk(0, q, torch.tensor([0, 8, -1], dtype=torch.int32, device=DEV), return_lse=True)
    with pytest.raises(RuntimeError, match="SHAPE"):
        c.check()
    assert torch.equal(out[0], good[0]) and (out[1:] == 0).all() and (lse[1:] == -math.inf).all()
    twice = c.attend_chunk(0, q[[1, 1]], torch.tensor([1, 1], dtype=torch.int32, device=DEV))
    assert torch.equal(twice[0], good[1]) and torch.equal(twice[1], good[1])
    c.check()
    c.table[2, 3] = 1 << 20
    c.attend_chunk(0, q)
    with pytest.raises(RuntimeError, match="SHAPE"):
        c.check()
    n = torch.tensor([70, 1000, -3], dtype=torch.int32, device=DEV)  # counts past M and below 0: as M and 0
    out = c.attend_chunk(0, q, None, n)
    assert torch.equal(out[:2], good[:2]) and (out[2] == 0).all()
    c.lens[1] = 20                                        # fewer tokens than the call names: the first see nothing
    out, lse = c.attend_chunk(0, q, return_lse=True)
    assert (out[1, :, :50] == 0).all() and (lse[1, :, :50] == -math.inf).all() and (out[1, :, 50:] != 0).any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_graph_streams_and_repeats(dtype):
    c = _cache(pages=400, blocks=100)
    _fill(c, [150, 99, 3000], seed=6)
    q = _query((3, 4, 90, 128), 8, dtype)
    want, lse = c.attend_chunk(0, q, return_lse=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    for k in range(4):                                    # two streams at once
        outs.append(c.attend_chunk(0, q))
        with torch.cuda.stream(side):
            outs.append(c.attend_chunk(0, q))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = c.attend_chunk(0, q)
        b, l2 = c.attend_chunk(0, q[:, :, :50], n_new=torch.full((3,), 50, dtype=torch.int32, device=DEV), return_lse=True)
    for _ in range(2):
        a.zero_()
        graph.replay()
        other = c.attend_chunk(0, q)
        torch.cuda.synchronize()
        assert torch.equal(a, want) and torch.equal(other, want)
    _check(c, q[:, :, :50], b, l2, [0, 1, 2], [50] * 3)


def test_pool_past_32_bits():
    import akv
    c = akv.Int4PagedCache(1, 130000, 8, 128, max_seqs=2, max_blocks=16, device=DEV)
    d = _cache(heads=8, seqs=2, blocks=16, pages=32)
    for x in (c, d):
        _fill(x, [300, 170], seed=9)
    for j in range(10):
        c.copy_pages([int(c.table[0, j])], [129980 + j])
        c.table[0, j] = 129980 + j
    q = _query((2, 16, 64, 128), 8, torch.bfloat16)
    assert torch.equal(c.attend_chunk(0, q), d.attend_chunk(0, q))
    c.check()


def test_large_scores():
    """Weights on one token, and scores far apart: nothing overflows."""
    c = _cache(heads=1)
    _fill(c, [400], scale=20.0)
    for dtype in (torch.float16, torch.bfloat16):
        q = _query((1, 4, 130, 128), 3, dtype, scale=10.0)
        out, lse = c.attend_chunk(0, q, return_lse=True)
        assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    q = _query((1, 4, 130, 128), 3, torch.float16, scale=10.0)
    out, lse = c.attend_chunk(0, q, return_lse=True)
    _check(c, q, out, lse, [0], [130])


def test_refusals():
    c = _cache()
    _fill(c, [40, 40])
    q = _query((2, 4, 30, 128), 1, torch.float16)
    for err, call in ((ValueError, lambda: c.attend_chunk(1, q)), (TypeError, lambda: c.attend_chunk(0, q.float())),
                      (ValueError, lambda: c.attend_chunk(0, q[:, :3])), (ValueError, lambda: c.attend_chunk(0, q[:, :, 0])),
                      (ValueError, lambda: c.attend_chunk(0, q[..., :64])), (RuntimeError, lambda: c.attend_chunk(0, q.cpu())),
                      (ValueError, lambda: c.attend_chunk(0, q, [0, 1, 2])), (ValueError, lambda: c.attend_chunk(0, q, None, [1])),
                      (ValueError, lambda: c.attend_chunk(0, q, out=q[:1])),
                      (ValueError, lambda: c.attend_chunk(0, q, out=q.bfloat16()))):
        with pytest.raises(err):
            call()
    assert c.attend_chunk(0, q[:0]).shape == (0, 4, 30, 128) and c.attend_chunk(0, q[:, :, :0]).shape == (2, 4, 0, 128)


@pytest.mark.parametrize("R,heads,rep,M", [(1100, 1, 1, 3), (700, 8, 1, 2)])
def test_more_rows_than_a_launch_lists(R, heads, rep, M):
    c = _cache(pages=R, heads=heads, dim=64, group=64, seqs=R, blocks=2)
    lens = [3 + i % 30 for i in range(R)]
    _fill(c, lens, seed=R)
    q = _query((R, heads * rep, M, 64), 3, torch.float16)
    out, lse = c.attend_chunk(0, q, return_lse=True)
    c.check()
    for i in (0, 511, 512, 513, 699, R - 1):
        r = torch.tensor([i], dtype=torch.int32, device=DEV)
        one, one_lse = c.attend_chunk(0, q[i:i + 1], r, return_lse=True)
        _check(c, q[i:i + 1], out[i:i + 1], lse[i:i + 1], [i], [M])
        assert torch.equal(one[0], out[i]) and torch.equal(one_lse[0], lse[i])


def test_long_chunk():
    """20,001 new tokens: a few of their queries against the formula."""
    n = 20001
    c = _cache(pages=640, heads=1, dim=64, group=64, seqs=1, blocks=640)
    _fill(c, [n], seed=5)
    q = _query((1, 2, n, 64), 6, torch.bfloat16)
    out, lse = c.attend_chunk(0, q, return_lse=True)
    c.check()
    for m in (0, 1, 127, 128, 9999, n - 2, n - 1):
        c.lens[0] = m + 1  # the query as the last of a row that ends with it
        _check(c, q[:, :, m:m + 1], out[:, :, m:m + 1], lse[:, :, m:m + 1], [0], [1])


def test_nothing_to_do():
    c = _cache(pages=8, blocks=4)
    _fill(c, [40, 5], seed=1)
    for shape in ((0, 4, 5, 128), (2, 4, 0, 128)):
        out, lse = c.attend_chunk(0, _query(shape, 1, torch.float16), torch.arange(shape[0], dtype=torch.int32, device=DEV),
                                  return_lse=True)
        assert out.shape == shape and lse.shape == shape[:3]
    c.check()
