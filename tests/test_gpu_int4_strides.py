"""GPU: append and read of tensors whose elements lie more than 2^31 apart."""
import pytest
import torch

import test_gpu_int4_cache as base

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("axis", [0, 1, 2])
def test_append_attend_with_offsets_past_32_bits(axis):
    """One axis of k, v and q strides by more than 2^31 elements (4 GB) in a buffer that holds little else."""
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("not enough free memory")
    step = (1 << 31) + 24
    shape = [2, 2, 3, 128]
    if axis == 2:
        shape[2] = 2
    small = torch.empty(shape).stride()
    stride = tuple(step if i == axis else s for i, s in enumerate(small))
    big = torch.empty((shape[axis] - 1) * step + 2 * 2 * 3 * 128, dtype=torch.float16, device=DEV)
    a, b = base._cache(heads=2), base._cache(heads=2)
    x = base._rand(shape, 1, torch.float16)
    far = big.as_strided(shape, stride)
    far.copy_(x)
    m = shape[2]
    for c, t in ((a, x), (b, far)):
        c.append(0, t, t, [0, 1], c.reserve([0, 1], m))
        c.check()
    assert torch.equal(a.buf, b.buf)
    want = a.attend(0, x, [0, 1])
    assert torch.equal(b.attend(0, far, [0, 1]), want)


def test_read_past_32_bits():
    """So many rows that the values read back are more than 2^31 elements."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("not enough free memory")
    import akv
    rows, tokens = 520, 4096                                         # x 8 heads x 128: 2.18e9 elements
    c = akv.Int4PagedCache(1, 140, 8, 128, max_seqs=rows, max_blocks=128, device=DEV)
    k = base._rand((1, 8, tokens, 128), 2, torch.float16)
    c.append(0, k, k, [0], c.reserve([0], tokens))
    c.fork(torch.zeros(rows - 1, dtype=torch.int32, device=DEV), torch.arange(1, rows, dtype=torch.int32, device=DEV))
    a, b = c.read(0, tokens)
    c.check()
    assert a.numel() > 1 << 31
    for i in (1, 255, 511, 512, 519):
        assert torch.equal(a[i], a[0]) and torch.equal(b[i], a[0])
    one, _ = c.read(0, tokens, [0])
    assert torch.equal(a[0], one[0])
