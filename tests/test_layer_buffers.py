"""A layer's buffers, without a GPU: what a captured `decode` writes is not a prefill's to outgrow."""
from types import SimpleNamespace

import pytest

import focr_hip
from focr_hip.layer import DecoderLayer
from test_binding_refusals import cuda


class Reached(Exception):
    pass


def stop(*_, **__):
    raise Reached


def test_factors_of_a_decode_have_a_buffer_of_their_own():
    layer, names = object.__new__(DecoderLayer), []
    layer.ctx, layer.n_heads, layer.capacity, layer.dim = SimpleNamespace(device=0), 16, 64, 192
    layer.prefix_len, layer.split = 0, None
    layer.qkv = SimpleNamespace(out_dim=2048, linear_ex=stop, prefill=stop)
    layer._buf = lambda name, shape: names.append(name)
    rotary = SimpleNamespace(ctx=layer.ctx, n_heads=16, factors=lambda positions, out: positions)
    for length, call in ((0, lambda h, rope: layer.prefill(h, rope, 0, 0)), (8, layer.decode)):
        layer.len, before = length, len(names)
        with pytest.raises(Reached):
            call(cuda(4, 192), focr_hip.RotaryRows(rotary, cuda(4, 3)))
        assert len(names) > before
    assert len(set(names)) == len(names), names
