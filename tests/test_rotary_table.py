"""The frequency table of `Rotary` and the contexts that read it, without a GPU."""
from types import SimpleNamespace

import pytest
import torch

import focr_hip


class Table:
    """Stands in for the frequencies on the device."""

    ndim, shape = 3, (2, 16, 32)

    def __init__(self, log):
        self.log = log

    def to(self, **_):
        self.log.append("copy")
        return self

    def contiguous(self):
        return self

    def data_ptr(self):
        return 4096


@pytest.fixture
def device(monkeypatch):
    """torch with one stream of a device; what the binding asks of it, in order."""
    log = []
    stream = SimpleNamespace(cuda_stream=7, synchronize=lambda: log.append("wait"))
    monkeypatch.setattr(focr_hip, "_torch", lambda: SimpleNamespace(
        as_tensor=lambda t: t, float32=torch.float32, cuda=SimpleNamespace(current_stream=lambda device: stream)))
    return log


@pytest.mark.parametrize("stream", [7, 8, None])  # torch's, another, the context's own
def test_the_table_is_complete_on_return(device, stream):
    # Whatever stream the rotary's own context is on: a cache of another context on another one
    # may be the first to read it.
    focr_hip.Rotary(Table(device), ctx=SimpleNamespace(handle=None, device=0, stream=stream))
    assert device == ["copy", "wait"]
