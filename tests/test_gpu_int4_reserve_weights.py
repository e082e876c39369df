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
