"""GPU: room is not taken for tokens whose weights cannot be kept."""
import pytest
import torch

from test_gpu_int4_weigh import DEV, _cache, _fill

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", ["shape", "type", "device", "strides"])
def test_reserve_refuses_before_it_takes_pages(bad):
    c = _cache(layers=2)
    _fill(c, [40, 70])
    good = c.weights
    c.weights = {"shape": good[:, :1].contiguous(), "type": good.double(), "device": good.cpu(),
                 "strides": good.transpose(1, 2).contiguous().transpose(1, 2)}[bad]
    state = c.page_state()
    with pytest.raises(ValueError):
        c.reserve([0, 1], [5, 100])
    assert torch.equal(c.page_state(), state)
    with pytest.raises(ValueError):
        c.fork([0], [5])
    assert torch.equal(c.page_state(), state)
    c.weights = good
    assert c.reserve([0, 1], [5, 100]).tolist() == [5, 100]
    assert c.lens.tolist()[:2] == [45, 170]


def test_weights_of_one_row_with_any_stride():
    """A dim of one has any stride in a contiguous tensor: the calls go by the sizes."""
    c = _cache(seqs=1, blocks=4, pages=8)
    c.weights = torch.zeros(128, device=DEV).as_strided((1, 1, 128), (0, 0, 1))
    assert c.weights.is_contiguous() and c.weights.stride(1) == 0
    c.weights += 3
    _fill(c, [70])
    assert c.weights[0, 0].tolist() == [0] * 70 + [3] * 58
    q = torch.randn(1, 4, 1, 128, device=DEV).half()
    _, lse = c.attend(0, q, return_lse=True)
    c.weigh(0, q, lse)
    assert abs(float(c.weights[0, 0, :70].sum()) - 4) < 1e-3
    assert c.evict(None, 64, first=4, recent=60).tolist() == [[*range(4), *range(10, 70)]]
    c.check()
