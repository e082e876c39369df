"""CPU: every entry of the 4-bit cache, and draft verification, launches with its tensors' GPU current.

A stream handle says nothing of its GPU where it is the default stream's (0): a launch goes to the GPU that is current.
The library and torch's notion of the current GPU are stood in for, so nothing is launched.
"""
import contextlib
import types

import pytest
import torch


class Gpu:
    """The current GPU (0 at first), and what each call of the library found as current."""

    def __init__(self, monkeypatch):
        from akv import _C
        self.now, self.calls = 0, []
        monkeypatch.setattr(_C, "current_device", lambda: self.now)
        monkeypatch.setattr(torch.cuda, "current_device", lambda: self.now)
        monkeypatch.setattr(torch.cuda, "device", self.device)
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)

    @contextlib.contextmanager
    def device(self, index):
        was, self.now = self.now, index if isinstance(index, int) else index.index
        try:
            yield
        finally:
            self.now = was

    def __getattr__(self, name):  # a library entry
        if not name.startswith("akv_"):
            raise AttributeError(name)

        def entry(*args):
            if name.endswith("_bytes"):
                return 64
            self.calls.append((name, self.now))
            return 0
        return entry


@pytest.fixture
def gpu(monkeypatch):
    from akv import _C
    g = Gpu(monkeypatch)
    monkeypatch.setattr(_C, "raw_stream", lambda index: 0)
    return g


def _cache(gpu, index):
    import akv
    c = akv.Int4PagedCache(2, 8, 2, 64, max_seqs=3, max_blocks=4, device="cpu")
    c._lib, c._dev_index = gpu, index
    return c


CALLS = {
    "append": lambda c: c.append(0, torch.zeros(1, 2, 1, 64).half(), torch.zeros(1, 2, 1, 64).half(), [0]),
    "read": lambda c: c.read(1, 2, [0]),
    "attend": lambda c: c.attend(0, torch.zeros(1, 4, 1, 64).half(), [0]),
    "reserve": lambda c: c.reserve([0], 1),
    "fork": lambda c: c.fork([0], [1]),
    "truncate": lambda c: c.truncate([0], [0]),
    "free": lambda c: c.free([0]),
    "compact": lambda c: c.compact(),
    "copy_pages": lambda c: c.copy_pages([0], [1]),
}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("index", [0, 1])
def test_the_cache_launches_on_its_own_gpu(gpu, name, index):
    c = _cache(gpu, index)
    gpu.calls.clear()
    CALLS[name](c)
    assert gpu.calls and all(now == index for _, now in gpu.calls)
    assert gpu.now == 0


def test_an_error_leaves_the_current_gpu(gpu):
    c = _cache(gpu, 1)
    with pytest.raises(ValueError):
        c.read(5, 1, [0])
    assert gpu.now == 0


class Fake:
    """A tensor's face, on a GPU that is not there."""

    def __init__(self, shape, dtype, index):
        self.shape, self.dtype, self.device = torch.Size(shape), dtype, torch.device("cuda", index)
        self._t = torch.empty(shape, device="meta")

    def dim(self):
        return len(self.shape)

    def stride(self):
        return self._t.stride()

    def contiguous(self):
        return self

    def data_ptr(self):
        return 4096


@pytest.mark.parametrize("index", [0, 1])
def test_verification_launches_on_its_tensors_gpu(gpu, monkeypatch, index):
    import akv
    from akv import _C, speculative
    monkeypatch.setattr(_C, "load", lambda: gpu)
    monkeypatch.setattr(speculative.torch, "empty_strided",
                        lambda shape, stride, dtype, device: Fake(shape, dtype, device.index))
    f32 = torch.float32
    akv.verify_draft(Fake((1, 3, 10), f32, index), Fake((1, 2, 10), f32, index), Fake((1, 2), torch.int64, index),
                     Fake((1, 2), f32, index), Fake((1,), f32, index))
    assert gpu.calls == [("akv_verify_draft", index)] and gpu.now == 0
    assert isinstance(akv, types.ModuleType)


@pytest.mark.parametrize("n_new", [-1, 1 << 31, (1 << 32) + 5])
def test_reserve_refuses_a_count_past_32_bits(gpu, n_new):
    """The entry takes a 32-bit count; a larger one would be cut to its low bits."""
    c = _cache(gpu, 0)
    gpu.calls.clear()
    with pytest.raises(ValueError):
        c.reserve([0], n_new)
    assert not gpu.calls
