"""GPU: the 4-bit paged cache (append, read, attention) against its formulas in 64 bits.

Append: per group z = fp16(min), s = fp16((max - z) / 15), c = rint((x - z) / s), value c*s + z.  The codes and the
stored pairs are compared bit for bit with numpy: the two fp16 roundings are part of the definition, and (x - z) and
the quotient of values that fp16 / bf16 inputs give round the same way in 32 and 64 bits except when the quotient
lies within 2^-22 of a tie, where either code is a nearest one (accepted).

Attention tolerances, derived before the first run.  With weights w_t (sum 1), values v_t = c_t s_t + z_t, out = sum
w_t v_t; the kernel may round each weight-times-scale to fp16 once, so |error| <= 2^-11 sum_t w_t s_t |c_t - 8| + the
output's own rounding 2^-11 |out| (fp16) or 2^-8 |out| (bf16) + fp32 sums (2^-20 of the largest |v|).
sum_t w_t s_t |c_t - 8| <= 8 max s <= 0.54 (max v - min v) of a group <= 1.1 vmax.  lse: fp32 logits, 2^-20 of the
largest |logit| + 1e-5.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _cache(layers=1, pages=64, heads=2, dim=128, group=None, seqs=8, blocks=16):
    import akv
    return akv.Int4PagedCache(layers, pages, heads, dim, group_size=group, max_seqs=seqs, max_blocks=blocks, device=DEV)


def _np_quantise(x, group):
    """Codes, scale and zero of float64 rows (..., D)."""
    x = np.nan_to_num(x, nan=0.0, posinf=65504.0, neginf=-65504.0).clip(-65504, 65504)
    g = x.reshape(*x.shape[:-1], -1, group)
    z = g.min(-1).astype(np.float16)
    s = ((g.max(-1) - z.astype(np.float64)) / 15).astype(np.float16)
    sd = s.astype(np.float64)[..., None]
    q = np.divide(g - z.astype(np.float64)[..., None], sd, out=np.zeros_like(g), where=sd > 0)
    return q.reshape(x.shape), s, z


def _fields(cache, layer, page, head, slot):
    """(K codes, V codes (D,), K pairs, V pairs (G, 2) fp16) of one token, numpy."""
    L = cache.layout
    rec = cache.buf[layer, page, head].cpu().numpy()
    D, G = cache.D, L.n_groups
    out = []
    for c, p in ((L.kc, L.kp), (L.vc, L.vp)):
        b = rec[c + slot * D // 2: c + (slot + 1) * D // 2]
        out.append(np.stack([b >> 4, b & 15], -1).reshape(-1))
        out.append(rec[p + slot * G * 4: p + (slot + 1) * G * 4].view(np.float16).reshape(G, 2))
    return out[0], out[2], out[1], out[3]


def _rand(shape, seed, dtype, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(shape, generator=g, device=DEV) * scale
    x[..., 3] *= 6
    return x.to(dtype)


@pytest.mark.parametrize("dim,group", [(64, 64), (64, 16), (128, 128), (128, 64), (128, 32), (256, 256), (256, 64)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_codes_and_pairs(dim, group, dtype):
    c = _cache(heads=3, dim=dim, group=group)
    rows = torch.tensor([2, 0, 5], dtype=torch.int32, device=DEV)
    n = torch.tensor([40, 1, 0], dtype=torch.int32, device=DEV)
    granted = c.reserve(rows, n)
    assert granted.tolist() == [40, 1, 0] and c.lens.tolist() == [1, 0, 40, 0, 0, 0, 0, 0]
    k, v = _rand((3, 3, 40, dim), 1, dtype), _rand((3, 3, 40, dim), 2, dtype)
    c.append(0, k, v, rows, granted)
    c.check()
    rk, rv = c.read(0, 40, rows, n_new=granted)
    for i, (row, cnt) in enumerate(((2, 40), (0, 1))):
        for t in range(cnt):
            page = int(c.table[row, t // 32])
            for h in range(3):
                kc, vc, kp, vp = _fields(c, 0, page, h, t % 32)
                for x, code, pair, back in ((k, kc, kp, rk), (v, vc, vp, rv)):
                    q, s, z = _np_quantise(x[i, h, t].double().cpu().numpy(), group)
                    np.testing.assert_array_equal(pair[:, 0], s)
                    np.testing.assert_array_equal(pair[:, 1], z)
                    near = np.abs(q - code) <= 0.5 * (1 + 2.0 ** -20)
                    assert near.all() or (code[~near] == q[~near].round().clip(0, 15)).all()
                    val = code.astype(np.float64) * np.repeat(pair[:, 0].astype(np.float64), group) + \
                        np.repeat(pair[:, 1].astype(np.float64), group)
                    got = back[i, h, t].double().cpu().numpy()
                    assert (np.abs(got - val) <= 2.0 ** -11 * np.abs(val) + 1e-7).all()
    assert (rk[2] == 0).all() and (rk[1, :, 1:] == 0).all()


def test_append_special_values():
    c = _cache(heads=1, dim=64, group=16)
    x = torch.zeros(1, 1, 4, 64, dtype=torch.float16, device=DEV)
    x[0, 0, 0, 0], x[0, 0, 0, 1], x[0, 0, 0, 2] = float("nan"), float("inf"), -float("inf")
    x[0, 0, 1] = 3.25                       # constant groups: scale 0, zero the value
    x[0, 0, 2, :16] = 1e-7                  # a range that rounds to nothing
    x[0, 0, 3] = torch.arange(64, device=DEV).half()
    g = c.reserve([0], 4)
    c.append(0, x, x, [0], g)
    k, v = c.read(0, 4, [0], n_new=g)
    c.check()
    assert torch.equal(k, v) and torch.isfinite(k).all()
    ref = x.nan_to_num(nan=0.0, posinf=65504.0, neginf=-65504.0)
    assert (k[0, 0, 1] == 3.25).all()
    # half a step of the group, plus the rounding of scale (15 steps of 2^-11), zero and output
    for t in range(4):
        r = ref[0, 0, t].double().view(4, 16)
        step = (r.amax(1) - r.amin(1)) / 15
        err = (k[0, 0, t].double().view(4, 16) - r).abs().amax(1)
        assert (err <= step * (0.5 + 15 * 2.0 ** -11) + 2.0 ** -10 * r.abs().amax(1) + 1e-7).all()


@pytest.mark.parametrize("dim,group", [(64, 16), (128, 32), (128, 128), (256, 128)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_unusual_tokens_among_ordinary_ones(dim, group, dtype):
    """NaN, infinities, a range past fp16's, a rounded-up minimum or a scale without its bits in single tokens:
    they get the formula's codes, and their neighbours what they get alone."""
    k = _rand((1, 2, 37, dim), 31, dtype)
    k[0, :, 20] = 0
    odd = k.clone()
    odd[0, 0, 2, 5] = float("nan")
    odd[0, 1, 7, 0], odd[0, 1, 7, group - 1] = float("inf"), -float("inf")
    odd[0, 0, 11, 9] = -float("inf")
    odd[0, 1, 13] *= 1e-6                   # the scale below fp16's normal range
    odd[0, 0, 18] = odd[0, 0, 18].abs() + 1.0000001e-7
    if dtype is torch.bfloat16:
        odd[0, 1, 22, 4], odd[0, 0, 30] = 1e5, 70000.0
        odd[0, 0, 26] = odd[0, 0, 26].abs() * 1e-5 + 1.1e-7  # minima that fp16 does not hold
    a, b, c = (_cache(heads=2, dim=dim, group=group) for _ in range(3))
    for cache, x in ((a, k), (b, odd)):
        cache.append(0, x, x, [0], cache.reserve([0], 37))
        cache.check()
    for t in range(37):
        c.append(0, odd[:, :, t:t + 1], odd[:, :, t:t + 1], [0], c.reserve([0], 1))
    assert torch.equal(b.buf, c.buf)        # in one call and one at a time
    same = (k == odd).all(-1)[0].cpu()
    for t in range(37):
        for h in range(2):
            f, g = _fields(b, 0, t // 32, h, t % 32), _fields(a, 0, t // 32, h, t % 32)
            if same[h, t]:
                assert all((x == y).all() for x, y in zip(f, g))
            q, s, z = _np_quantise(odd[0, h, t].double().cpu().numpy(), group)
            np.testing.assert_array_equal(f[2][:, 0], s)
            np.testing.assert_array_equal(f[2][:, 1], z)
            near = np.abs(q - f[0]) <= 0.5 * (1 + 2.0 ** -20)
            assert near.all() or (f[0][~near] == q[~near].round().clip(0, 15)).all()
            assert (f[0] == f[1]).all() and (f[2] == f[3]).all()


@pytest.mark.parametrize("layout", ["token_major", "odd_stride", "odd_offset", "last_dim"])
def test_append_strides(layout):
    a, b = _cache(heads=2), _cache(heads=2)
    k, v = _rand((2, 2, 7, 128), 3, torch.float16), _rand((2, 2, 7, 128), 4, torch.float16)
    if layout == "token_major":
        ks, vs = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
    elif layout == "odd_stride":
        big = torch.zeros(2, 2, 7, 131, dtype=torch.float16, device=DEV)
        ks, vs = big[..., :128], big.clone()[..., :128]
        ks.copy_(k), vs.copy_(v)
    elif layout == "odd_offset":
        flat = torch.zeros(2, k.numel() + 1, dtype=torch.float16, device=DEV)
        ks, vs = flat[0, 1:].view(k.shape), flat[1, 1:].view(k.shape)
        ks.copy_(k), vs.copy_(v)
    else:
        ks, vs = (x.transpose(2, 3).contiguous().transpose(2, 3) for x in (k, v))
    for c, (kk, vv) in ((a, (k, v)), (b, (ks, vs))):
        g = c.reserve([0, 1], 7)
        c.append(0, kk, vv, [0, 1], g)
        c.check()
    assert torch.equal(a.buf, b.buf)


def test_append_writes_only_its_slots():
    c = _cache(layers=2, heads=2)
    c.buf.random_(0, 256)
    g = c.reserve([1], 33)
    before = c.buf.clone()
    k = _rand((1, 2, 33, 128), 5, torch.float16)
    c.append(1, k, k, [1], g)
    c.check()
    assert torch.equal(c.buf[0], before[0])
    p = c.table[1, :2].tolist()
    others = [i for i in range(c.n_pages) if i not in p]
    assert torch.equal(c.buf[1, others], before[1, others])
    L = c.layout
    for off, width in ((L.kc, 64), (L.vc, 64), (L.kp, 4), (L.vp, 4)):  # the second page holds one token
        a = c.buf[1, p[1], :, off + width: off + 32 * width]
        assert torch.equal(a, before[1, p[1], :, off + width: off + 32 * width])


def _reference(c, layer, q, rows, n_new, scale):
    """fp64 attention, its lse and the bound max|v| of each row, from the values the cache stands for."""
    R, Hq, M, D = q.shape
    rep = Hq // c.H
    out = torch.zeros(R, Hq, M, D, dtype=torch.float64, device=DEV)
    lse = torch.full((R, Hq, M), -math.inf, dtype=torch.float64, device=DEV)
    vmax = torch.zeros(R, 1, 1, 1, dtype=torch.float64, device=DEV)
    xmax = torch.zeros(R, 1, 1, dtype=torch.float64, device=DEV)
    L, G = c.layout, c.layout.n_groups
    for i in range(R):
        row, new = int(rows[i]), min(int(n_new[i]), M)
        n = int(c.lens[row])
        if n == 0:
            continue
        pages = c.table[row, :(n + 31) // 32].long()
        rec = c.buf[layer, pages].transpose(0, 1)  # (H, blocks, rec)
        kv = []
        for co, po in ((L.kc, L.kp), (L.vc, L.vp)):
            b = rec[..., co:co + 16 * D].reshape(c.H, -1, D // 2)[:, :n]
            p = rec[..., po:po + 128 * G].contiguous().view(torch.float16).reshape(c.H, -1, G, 2)[:, :n].double()
            code = torch.stack([b >> 4, b & 15], -1).flatten(-2).double().unflatten(-1, (G, -1))
            kv.append((code * p[..., :1] + p[..., 1:]).flatten(-2))
        vmax[i] = kv[1].abs().max()
        for m in range(new):
            see = n - new + m + 1
            if see <= 0:
                continue
            for h in range(Hq):
                x = kv[0][h // rep, :see] @ q[i, h, m].double() * scale
                xmax[i] = torch.maximum(xmax[i], x.abs().max())
                lse[i, h, m] = torch.logsumexp(x, 0)
                out[i, h, m] = torch.softmax(x, 0) @ kv[1][h // rep, :see]
    return out, lse, vmax, xmax


def _check(c, layer, q, rows, n_new, scale=None, out=None):
    rows_t = None if rows is None else torch.tensor(rows, dtype=torch.int32, device=DEV)
    R, M = q.shape[0], q.shape[2]
    nn_t = None if n_new is None else torch.tensor(n_new, dtype=torch.int32, device=DEV)
    got, lse = c.attend(layer, q, rows_t, nn_t, sm_scale=scale, out=out, return_lse=True)
    c.check()
    ref, rlse, vmax, xmax = _reference(c, layer, q, range(R) if rows is None else rows, n_new or [M] * R,
                                       1 / math.sqrt(c.D) if scale is None else scale)
    eps = 2.0 ** -11 if q.dtype == torch.float16 else 2.0 ** -8
    err = (got.double() - ref).abs()
    assert (err <= eps * ref.abs() + (1.1 * 2.0 ** -11 + 2.0 ** -20) * vmax).all(), float(err.max())
    assert torch.equal(torch.isfinite(lse), torch.isfinite(rlse))
    fin = torch.isfinite(rlse)
    assert ((lse.double() - rlse).abs()[fin] <= (2.0 ** -20 * xmax + 1e-5).expand_as(lse)[fin]).all()
    return got, lse


def _filled(lens, dim=128, group=None, heads=2, seed=0, dtype=torch.float16, kscale=1.0, vscale=1.0, layers=1, junk=True):
    """A cache whose row i holds lens[i] tokens on shuffled pages; unused bytes are all ones (NaN scales)."""
    blocks = max(1, max((n + 31) // 32 for n in lens)) + 1
    pages = sum((n + 31) // 32 for n in lens) + 5
    c = _cache(layers, pages, heads, dim, group, len(lens), blocks)
    if junk:
        c.buf.fill_(255)
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).int()
    table, at = torch.full((len(lens), blocks), -1, dtype=torch.int32), 0
    for i, n in enumerate(lens):
        nb = (n + 31) // 32
        table[i, :nb] = perm[at:at + nb]
        at += nb
    c.load_state(c.buf.clone(), table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV))
    M = max(max(lens), 1)
    for layer in range(layers):
        k = _rand((len(lens), heads, M, dim), seed + 10 + layer, dtype, kscale)
        v = _rand((len(lens), heads, M, dim), seed + 20 + layer, dtype, vscale)
        c.append(layer, k, v, None, torch.tensor(lens, dtype=torch.int32, device=DEV))
    c.check()
    return c


LENS = [0, 1, 31, 32, 33, 64, 95, 257, 1000]


@pytest.mark.parametrize("dim,group", [(64, 64), (64, 32), (64, 16), (128, 128), (128, 64), (128, 32),
                                       (256, 256), (256, 128), (256, 64)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attend_single_token(dim, group, dtype):
    c = _filled(LENS, dim, group)
    _check(c, 0, _rand((len(LENS), 8, 1, dim), 7, dtype), None, None)


@pytest.mark.parametrize("rep,m", [(1, 1), (1, 2), (3, 3), (4, 5), (7, 1), (8, 4), (5, 7), (6, 12), (2, 33)])
@pytest.mark.parametrize("dim,group", [(128, 128), (128, 32), (64, 32), (256, 128)])
def test_attend_drafted_tokens(rep, m, dim, group):
    c = _filled(LENS, dim, group)
    g = torch.Generator().manual_seed(m)
    n_new = torch.randint(0, m + 1, (len(LENS),), generator=g).tolist()
    n_new[-1] = m
    _check(c, 0, _rand((len(LENS), 2 * rep, m, dim), 8, torch.bfloat16), None, n_new)
    _check(c, 0, _rand((len(LENS), 2 * rep, m, dim), 9, torch.float16), None, None)


@pytest.mark.parametrize("n", [4095, 4096, 16385, 70001])
def test_attend_long(n):
    c = _filled([n, 17, n // 3], 128, 64, heads=1)
    _check(c, 0, _rand((3, 4, 2, 128), 11, torch.float16), None, [2, 1, 2])


def test_attend_many_rows_few_heads_and_one_head_pair():
    c = _filled([40 + 13 * i for i in range(70)], 128, 128, heads=1)
    _check(c, 0, _rand((70, 1, 1, 128), 12, torch.float16), None, None)


@pytest.mark.parametrize("kscale,vscale", [(1e-3, 1e-3), (1.0, 300.0), (20.0, 1.0), (1.0, 1e-4), (0.0, 1.0)])
def test_attend_magnitudes(kscale, vscale):
    c = _filled([300, 33], 128, 64, kscale=kscale, vscale=vscale)
    _check(c, 0, _rand((2, 4, 3, 128), 13, torch.float16, 2.0), None, None)


def test_attend_values_of_very_different_size():
    """One token's values dwarf the others'."""
    c = _filled([200], 128, 64, vscale=1e-3)
    k, v = _rand((1, 2, 1, 128), 14, torch.float16), _rand((1, 2, 1, 128), 15, torch.float16, 1000.0)
    g = c.reserve([0], 1)
    c.append(0, k, v, [0], g)
    _check(c, 0, _rand((1, 4, 1, 128), 16, torch.float16), None, None)


def test_attend_large_queries():
    """Queries near fp16's and beyond fp16's range (bf16)."""
    c = _filled([130], 128, 128, kscale=1e-3)
    q = _rand((1, 4, 1, 128), 17, torch.float16, 5000.0).clamp(-60000, 60000)
    _check(c, 0, q, None, None, scale=1e-3)
    q = _rand((1, 4, 1, 128), 18, torch.bfloat16, 1e6)
    _check(c, 0, q, None, None, scale=1e-6)
    q = torch.zeros(1, 4, 1, 128, dtype=torch.float16, device=DEV)
    _check(c, 0, q, None, None)


def test_attend_rows_order_strides_and_out():
    c = _filled(LENS, 128, 64, layers=2)
    rows = [8, 2, 5, 0]
    q = _rand((4, 3, 8, 128), 19, torch.float16).transpose(1, 2)      # token-major storage
    _check(c, 1, q, rows, [3, 1, 2, 0])
    big = torch.zeros(4, 8, 3, 129, dtype=torch.float16, device=DEV)  # odd strides
    big[..., 1:] = q
    out = torch.full((4, 3, 8, 130), 7.0, dtype=torch.float16, device=DEV)[..., :128].transpose(1, 2)
    got, _ = _check(c, 1, big[..., 1:], rows, [3, 1, 2, 0], out=out)
    assert got.data_ptr() == out.data_ptr()
    o3 = c.attend(1, q[:, :, 0], torch.tensor(rows, dtype=torch.int32, device=DEV))
    assert o3.shape == (4, 8, 128)
    # more new tokens than the row holds: the first queries stand before its start
    _check(c, 1, _rand((1, 8, 3, 128), 20, torch.float16), [1], [3])


def test_attend_same_pages_in_two_rows_and_repeated_calls():
    c = _filled([100, 0], 128, 128)
    c.fork([0], [1])
    q = _rand((1, 4, 1, 128), 21, torch.float16)
    a = c.attend(0, q, [0])
    b = c.attend(0, q, [1])
    d = c.attend(0, q, [0])
    c.check()
    assert torch.equal(a, b) and torch.equal(a, d)


def test_attend_shapes_in_turn_on_one_workspace():
    """Calls of very different shapes share the stream's scratch: no call may see what another left."""
    c = _filled([1500, 700, 33, 1], 128, 128, heads=2)
    shapes = [(4, 2, 1), (1, 8, 2), (4, 16, 3), (2, 4, 12), (4, 2, 1), (1, 2, 1), (4, 16, 8)]
    for i, (r, hq, m) in enumerate(shapes * 2):
        _check(c, 0, _rand((r, hq, m, 128), 30 + i, torch.float16), None, None)


def test_attend_on_another_stream_and_in_a_graph():
    c = _filled([500, 37], 128, 64)
    q = _rand((2, 4, 2, 128), 22, torch.float16)
    ref = c.attend(0, q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = c.attend(0, q)
    s.synchronize()
    assert torch.equal(got, ref)
    rows, n = torch.tensor([0, 1], dtype=torch.int32, device=DEV), torch.tensor([2, 2], dtype=torch.int32, device=DEV)
    k = _rand((2, 2, 2, 128), 23, torch.float16)
    lens = c.lens.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        granted = c.reserve(rows, n)
        c.append(0, k, k, rows, granted)
        out = c.attend(0, q, rows, granted)
        c.truncate(rows, lens)
    state = c.page_state()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    c.check()
    assert torch.equal(c.page_state(), state)
    g2 = c.reserve(rows, n)
    c.append(0, k, k, rows, g2)
    assert torch.equal(out, c.attend(0, q, rows, g2))


def test_bad_rows_and_pages_set_status():
    c = _filled([64, 64], 128, 128)
    q = _rand((2, 2, 1, 128), 24, torch.float16)
    out = c.attend(0, q, [0, 9])
    with pytest.raises(RuntimeError, match="AKV_ERR_SHAPE"):
        c.check()
    assert (out[1] == 0).all() and torch.isfinite(out).all()
    c.table[1, 1] = 10 ** 6
    before = c.buf.clone()
    c.attend(0, q)
    with pytest.raises(RuntimeError, match="AKV_ERR_SHAPE"):
        c.check()
    k = _rand((2, 2, 1, 128), 25, torch.float16)
    c.append(0, k[1:], k[1:], [1])
    with pytest.raises(RuntimeError, match="AKV_ERR_SHAPE"):
        c.check()
    assert torch.equal(c.buf, before)
    c.read(0, 3, [7])
    with pytest.raises(RuntimeError, match="AKV_ERR_SHAPE"):
        c.check()


def test_refusals():
    import akv
    c = _filled([64, 64], 128, 128)
    q = _rand((2, 4, 1, 128), 26, torch.float16)
    k = _rand((2, 2, 1, 128), 27, torch.float16)
    for bad in (dict(head_dim=96), dict(head_dim=128, group_size=48), dict(head_dim=128, group_size=16)):
        with pytest.raises(RuntimeError, match="AKV_ERR_SHAPE"):
            akv.Int4PagedCache(1, 4, 2, device=DEV, **bad)
    with pytest.raises(ValueError):
        akv.Int4PagedCache(1, 0, 2, 128, device=DEV)
    with pytest.raises(ValueError):
        c.attend(1, q)
    with pytest.raises(ValueError):
        c.attend(0, q[:, :3])
    with pytest.raises(ValueError):
        c.attend(0, q[..., :64])
    with pytest.raises(TypeError):
        c.attend(0, q.float())
    with pytest.raises(RuntimeError):
        c.attend(0, q.cpu())
    with pytest.raises(ValueError):
        c.attend(0, q, torch.tensor([0, 1], device=DEV))            # int64 rows
    with pytest.raises(ValueError):
        c.attend(0, q, [0])
    with pytest.raises(ValueError):
        c.attend(0, q, out=torch.empty_like(q, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        c.attend(0, _rand((3, 4, 1, 128), 1, torch.float16))         # three rows, two sequences
    with pytest.raises(TypeError):
        c.append(0, k, k.bfloat16())
    with pytest.raises(ValueError):
        c.append(0, k, k[:, :, :, :64])
    with pytest.raises(TypeError):
        c.read(0, 1, dtype=torch.float32)
    with pytest.raises(ValueError):
        c.load_state(c.buf, c.table[:, :1], c.lens)
    bad = c.table.clone()
    bad[0, 0] = c.n_pages
    with pytest.raises(ValueError):
        c.load_state(c.buf, bad, c.lens)
    assert c.attend(0, q[:0], []).shape == (0, 4, 1, 128)
    assert c.attend(0, q[:, :, :0]).shape == (2, 4, 0, 128)
    c.check()


def test_state_refusals():
    c = _filled([64, 40], 128, 128)
    state = c.page_state()
    for bad in (-1, c.max_blocks * 32 + 1):
        lens = c.lens.clone()
        lens[1] = bad
        with pytest.raises(ValueError):
            c.load_state(c.buf, c.table, lens)
    for bad in (state[:1], state[:-1], state.long()):
        with pytest.raises(ValueError):
            c.set_page_state(bad)
    assert torch.equal(c.page_state(), state)
    c.set_page_state(state)
    assert torch.equal(c.page_state(), state)
