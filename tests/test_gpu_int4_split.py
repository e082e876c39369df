"""GPU: attention over the 4-bit cache where units are cut over several CTAs, merged in either way, or launched in
several parts.  Formula and tolerances are those of the cache's other attention tests."""
import math

import pytest
import torch

import test_gpu_int4_cache as base

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
SHAPES = [(64, 64), (64, 32), (64, 16), (128, 128), (128, 64), (128, 32), (256, 256), (256, 128), (256, 64)]


@pytest.mark.parametrize("dim,group", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_one_token(dim, group, dtype):
    lens = [0, 1025, 3001, 31, 1500]
    c = base._filled(lens, dim, group)
    base._check(c, 0, base._rand((len(lens), 8, 1, dim), 7, dtype), None, None)


@pytest.mark.parametrize("rep,m", [(1, 2), (3, 3), (4, 5), (7, 1), (2, 17)])
@pytest.mark.parametrize("dim,group", SHAPES)
def test_drafted_tokens(rep, m, dim, group):
    lens = [1025, 0, 2047, 64]
    c = base._filled(lens, dim, group)
    n_new = [m, m, max(m - 1, 1), m]
    base._check(c, 0, base._rand((len(lens), 2 * rep, m, dim), 8, torch.bfloat16), None, n_new)
    base._check(c, 0, base._rand((len(lens), 2 * rep, m, dim), 9, torch.float16), None, None)


@pytest.mark.parametrize("dim,group", SHAPES)
@pytest.mark.parametrize("rep,m", [(1, 1), (4, 3), (7, 2)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_merged_by_a_second_kernel(dim, group, rep, m, dtype):
    """A long table: a unit may have more parts than its last CTA merges by itself."""
    blocks = 8200
    c = base._cache(1, 400, 2, dim, group, 3, blocks)
    lens = torch.tensor([6000, 0, 3333], dtype=torch.int32, device=DEV)
    c.reserve(None, lens)
    k, v = base._rand((3, 2, 6000, dim), 1, torch.float16), base._rand((3, 2, 6000, dim), 2, torch.float16)
    c.append(0, k, v, None, lens)
    base._check(c, 0, base._rand((3, 2 * rep, m, dim), 3, dtype), None, [m, m, max(m - 1, 1)])


@pytest.mark.parametrize("dim,group,dtype", [(64, 64, torch.float16), (128, 32, torch.bfloat16),
                                             (128, 128, torch.float16)])
def test_more_rows_than_one_launch_holds(dim, group, dtype):
    """2,500 (row, row tile) pairs: three launches, short rows and some long ones."""
    rows = 1250
    lens = [(37 * i) % 90 for i in range(rows)]
    lens[3], lens[700], lens[1249] = 1100, 1300, 1500
    c = base._filled(lens, dim, group, heads=1)
    pick = [0, 1, 3, 511, 512, 513, 699, 700, 701, 1023, 1024, 1025, 1248, 1249]
    q = base._rand((rows, 8, 4, dim), 5, dtype)
    n_new = torch.tensor([(i % 4) + 1 for i in range(rows)], dtype=torch.int32, device=DEV)
    out, lse = c.attend(0, q, None, n_new, return_lse=True)
    c.check()
    one, lone = base._check(c, 0, q[pick], pick, n_new[pick].tolist())
    # the same rows in a call of their own are cut otherwise, but have the same values: twice the bound apart
    ref, rlse, vmax, xmax = base._reference(c, 0, q[pick], pick, n_new[pick].tolist(), 1 / math.sqrt(dim))
    eps = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8
    assert ((out[pick].double() - ref).abs() <= eps * ref.abs() + (1.1 * 2.0 ** -11 + 2.0 ** -20) * vmax).all()
    fin = torch.isfinite(rlse)
    assert torch.equal(torch.isfinite(lse[pick]), fin)
    assert ((lse[pick].double() - rlse).abs()[fin] <= (2.0 ** -20 * xmax + 1e-5).expand_as(rlse)[fin]).all()
    # every row: queries past n_new and rows without a token are zero, the others are not
    past = torch.arange(4, device=DEV)[None] >= n_new[:, None]
    before = torch.arange(4, device=DEV)[None] < (n_new - c.lens)[:, None]
    none = (past | before)[:, None].expand(rows, 8, 4)
    assert (out[none] == 0).all() and (lse[none] == -math.inf).all()
    assert torch.isfinite(lse[~none]).all() and (out[~none] != 0).any(-1).all()


def test_256_sequences():
    lens = [33 + 7 * (i % 40) for i in range(256)]
    lens[100] = 1200
    c = base._filled(lens, 128, 128, heads=2)
    base._check(c, 0, base._rand((256, 2, 1, 128), 6, torch.float16), None, None)


def test_more_units_than_one_launch_counts():
    """64 KV heads and 300 rows: 19,200 units."""
    lens = [(11 * i) % 50 for i in range(300)]
    lens[299] = 1100
    c = base._filled(lens, 64, 64, heads=64)
    q = base._rand((300, 64, 1, 64), 7, torch.float16)
    pick = [0, 1, 255, 256, 257, 298, 299]
    out = c.attend(0, q)
    ref, _, vmax, _ = base._reference(c, 0, q[pick], pick, [1] * len(pick), 1 / 8)
    c.check()
    assert ((out[pick].double() - ref).abs() <= 2.0 ** -11 * ref.abs() + (1.1 * 2.0 ** -11 + 2.0 ** -20) * vmax).all()


@pytest.mark.parametrize("dim,group,dtype", [(64, 16, torch.bfloat16), (256, 256, torch.float16)])
def test_on_another_stream_and_in_a_graph(dim, group, dtype):
    c = base._filled([1500, 1037], dim, group)
    q = base._rand((2, 4, 5, dim), 22, dtype)
    ref = c.attend(0, q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = c.attend(0, q)
    s.synchronize()
    assert torch.equal(got, ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.attend(0, q)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref)
    c.check()
