"""The frequency table of `Rotary` and the contexts that read it, without a GPU."""
from types import SimpleNamespace

import pytest
import torch

import focr_hip
from test_binding_refusals import cuda
from test_served_abi import pages


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
        as_tensor=lambda t: t, float32=torch.float32,
        cuda=SimpleNamespace(current_stream=lambda device: stream, is_current_stream_capturing=lambda: "capture" in log)))
    return log


@pytest.mark.parametrize("stream", [7, 8, None])  # torch's, another, the context's own
def test_the_table_is_complete_on_return(device, stream):
    # Whatever stream the rotary's own context is on: a cache of another context on another one
    # may be the first to read it.
    focr_hip.Rotary(Table(device), ctx=SimpleNamespace(handle=None, device=0, stream=stream))
    assert device == ["copy", "wait"]


def context(device, stream, name="ctx"):
    return SimpleNamespace(handle=None, device=0, stream=stream, sync=lambda: device.append(name))


@pytest.mark.parametrize("stream,waits", [(7, []), (8, ["ctx"]), (None, ["ctx"])])
def test_the_table_is_kept_until_other_streams_have_read_it(device, stream, waits):
    # Its memory goes to the next tensor of torch's stream.
    rotary = focr_hip.Rotary(Table(device), ctx=context(device, stream))
    device.clear()
    del rotary
    assert device == waits


@pytest.mark.parametrize("stream", [7, 9])
def test_a_cache_of_another_context_is_waited_for(device, stream, monkeypatch):
    monkeypatch.setattr(focr_hip, "lib", lambda: SimpleNamespace(focr_kv_pages_qkv_rows_at=lambda *_: 0))
    kv, x = pages(), cuda(2, 32 * 64)
    kv.ctx = context(device, stream, "cache")
    rotary = focr_hip.Rotary(Table(device), ctx=context(device, 7))
    for _ in range(2):
        kv.qkv_rows(x, rotary.at(cuda(2, 2)), cuda(2, dtype=torch.int32), q=cuda(2, 16, 64))
    device.clear()
    del rotary
    assert device == (["cache"] if stream != 7 else [])


@pytest.mark.parametrize("stream", [7, 8])
def test_a_capture_is_not_waited_in(device, stream, monkeypatch):
    # The table stays instead, where another stream may read it.
    monkeypatch.setattr(focr_hip, "_kept_tables", [])
    table = Table(device)
    rotary = focr_hip.Rotary(table, ctx=context(device, stream))
    device[:] = ["capture"]
    del rotary
    assert device == ["capture"] and focr_hip._kept_tables == ([table] if stream == 8 else [])
