"""GPU: the codes that append writes are those of the true division, in 32 bits, bit for bit.

scale = fp16((max - zero) / 15) and code = clamp(rint((x - zero) / scale), 0, 15) are IEEE divisions of fp32 numbers.
The kernel takes the quotient by a reciprocal and one correction; here it meets every positive scale that fp16 has up
to the largest a group can get, with numerators at, next to and between the half steps, where a quotient off by a
unit in its last place gives another code.
"""
import numpy as np
import pytest
import torch

import test_gpu_int4_cache as base

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _codes(x, group):
    """append's (codes, scales, zeros) of rows x (N, D) of any type, numpy."""
    import akv
    n, dim = x.shape
    c = akv.Int4PagedCache(1, (n + 31) // 32, 1, dim, group_size=group, max_seqs=1, max_blocks=(n + 31) // 32,
                           device=DEV)
    x = x[None, None].to(DEV)
    c.append(0, x, x, [0], c.reserve([0], n))
    c.check()
    L, G = c.layout, c.layout.n_groups
    rec = c.buf[0, c.table[0].long(), 0]
    b = rec[:, L.kc:L.kc + 16 * dim].reshape(-1, dim // 2)[:n]
    p = rec[:, L.kp:L.kp + 128 * G].contiguous().view(torch.float16).reshape(-1, G, 2)[:n]
    return torch.stack([b >> 4, b & 15], -1).flatten(1).cpu().numpy(), p[..., 0].cpu().numpy(), p[..., 1].cpu().numpy()


def _formula(x, group):
    """The same by numpy's division of float32 (values past fp16's range count as its ends)."""
    g = x.float().numpy().clip(-65504, 65504).reshape(x.shape[0], -1, group)
    z = g.min(-1).astype(np.float16)
    zf = z.astype(np.float32)
    s = ((g.max(-1) - zf) / np.float32(15)).astype(np.float16)
    sf = s.astype(np.float32)[..., None]
    q = np.divide(g - zf[..., None], sf, out=np.zeros_like(g), where=sf > 0)
    assert q.dtype == np.float32
    return np.rint(q).clip(0, 15).astype(np.uint8).reshape(x.shape), s, z


def _same(x, group):
    for a, b in zip(_codes(x, group), _formula(x, group)):
        bad = np.argwhere(a != b)
        assert not len(bad), (len(bad), bad[:3].tolist(), a[tuple(bad[0])], b[tuple(bad[0])])


def _near(v, dtype, rng, steps):
    """v rounded to dtype and its neighbours a few units in the last place away."""
    t = torch.from_numpy(v).to(dtype)
    up = (t.view(torch.int16) + torch.from_numpy(rng.integers(-steps, steps + 1, v.shape).astype(np.int16)))
    near = up.view(dtype)
    return torch.where(torch.isfinite(near.float()) & (near.float().sign() == t.float().sign()), near, t)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("zero", [0.0, 1.0, -0.37, -300.0, -9000.0])
def test_every_scale(dtype, zero):
    """Groups from `zero` to zero + 15 s for every positive fp16 s that stays in range: half steps and around them."""
    rng = np.random.default_rng(int(abs(zero)))
    s = np.arange(1, 0x7C00, dtype=np.uint16).view(np.float16).astype(np.float64)
    lo = float(torch.tensor(zero).to(dtype))
    s = s[lo + 15 * s <= 65504]
    k = np.arange(128)
    rows = []
    for shift in range(2):
        v = lo + s[:, None] * ((k % 15) + 0.5)[None]
        x = _near(v, dtype, rng, shift * 3)
        x = torch.where(x.float() < lo, torch.tensor(lo, dtype=dtype), x)
        top = torch.from_numpy(lo + 15 * s).to(dtype)
        x = torch.minimum(x.float(), top.float()[:, None]).to(dtype)
        x[:, 0], x[:, 64] = lo, lo
        x[:, 1], x[:, 65] = top, top
        rows.append(x)
    _same(torch.cat(rows), 64)
    _same(torch.cat(rows), 128)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,group", [(64, 16), (128, 32), (256, 256)])
def test_random_bits(dtype, dim, group):
    """Rows of every magnitude, and rows whose magnitudes differ within a group."""
    rng = np.random.default_rng(dim + group)
    n = 40000
    mag = 2.0 ** rng.uniform(-24, 15.9, (n, 1))
    x = rng.standard_normal((n, dim)) * mag
    x[::3] *= 2.0 ** rng.uniform(-12, 0, (len(x[::3]), dim))
    x[1::5] += rng.uniform(-2, 2, (len(x[1::5]), 1)) * mag[1::5]
    _same(torch.from_numpy(x).to(dtype), group)
