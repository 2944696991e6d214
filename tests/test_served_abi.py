"""Rotary factors, the row step from positions, attention over a shared prefix and rules on
logits, without a GPU: null arguments are errors, and what the binding refuses by itself."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import focr_hip
from test_binding_refusals import cuda, refused


def test_null_arguments_are_errors_not_crashes():
    lib = focr_hip.lib()
    assert lib.focr_rotary_factors(None, None, 1, 1, None, 16, 64, None) == -1
    assert "null" in lib.focr_last_error().decode()
    assert lib.focr_kv_pages_qkv_rows_at(None, None, None, 1, None, 1, None, None, None, 1, None) == -1
    assert lib.focr_kv_pages_attention_shared(None, None, None, 1, None, None, 1, 64, 0, 16, None, None) == -1
    assert lib.focr_logits_select(None, None, 1, 8, None, None, 0, 0, None, 0, None, None, 0, 0, None, 0, 0, None, None) == -1


CTX = SimpleNamespace(handle=None, device=0)


def i32(*shape, **kw):
    return cuda(*shape, dtype=torch.int32, **kw)


@pytest.mark.parametrize("shape", [(5, 16, 32), (0, 16, 32), (2, 16, 31), (16, 32)])
def test_frequencies_of_other_shapes(shape):
    refused(-2, lambda: focr_hip.Rotary(np.ones(shape, np.float32), ctx=CTX))


def test_positions():
    rotary = object.__new__(focr_hip.Rotary)
    rotary.ctx, rotary.axes, rotary.n_heads, rotary._table = CTX, 2, 16, 4096
    for p in (cuda(4, 3), cuda(8)):
        refused(-2, lambda: rotary.factors(p, out=cuda(4, 16, 32, 2)))
        refused(-2, lambda: rotary.at(p))
    refused(-2, lambda: rotary.factors(cuda(4, 2), out=cuda(3, 16, 32, 2)))
    refused(-2, lambda: rotary.factors(cuda(4, 2, dtype=torch.int32), out=cuda(4, 16, 32, 2)))
    refused(-1, lambda: rotary.factors(cuda(4, 2, device=1), out=cuda(4, 16, 32, 2)))
    refused(-2, lambda: rotary.factors(cuda(4, 2, contiguous=False), out=cuda(4, 16, 32, 2)))


def pages():
    kv = object.__new__(focr_hip.KvPages)
    kv.ctx, kv.handle, kv.n_heads, kv.n_kv_heads, kv.key_heads, kv.n_seqs = CTX, None, 16, 8, 8, 2
    kv._float, kv._int, kv._device = torch.float32, torch.int32, 0
    return kv


def test_row_steps_from_positions():
    kv, lens = pages(), i32(2)
    at = lambda p, heads=16, device=0: focr_hip.RotaryRows(SimpleNamespace(ctx=SimpleNamespace(device=device), axes=2, n_heads=heads, _table=4096), p)  # noqa: E731
    for code, rope in ((-2, at(cuda(3, 2))), (-2, at(cuda(2, 2), heads=8)), (-1, at(cuda(2, 2), device=1)),
                       (-2, at(cuda(2, 2, dtype=torch.float64))), (-1, at(cuda(2, 2, device=1)))):
        refused(code, lambda: kv.qkv_rows(cuda(2, 32 * 64), rope, lens, q=cuda(2, 16, 64)))


def test_shared_prefixes():
    kv, q, lens = pages(), cuda(2, 16, 64), i32(2)
    for shared, prefix in ((-16, 0), (16, 2), (16, -1)):
        refused(-2, lambda: kv.attention_shared(q, lens, 64, shared, prefix, out=q))
    refused(-2, lambda: kv.attention_shared(q, cuda(2), 64, 16, out=q))
    refused(-2, lambda: kv.attention_shared(q, lens, 0, 16, out=q))
    refused(-2, lambda: kv.attention_shared(q, lens, 64, 16, sinks=cuda(8), out=q))


def test_rules_of_other_sizes():
    R, x, to = focr_hip.LogitRules, cuda(4, 100), i32(4)
    history = dict(history=i32(4, 9), lengths=i32(4))
    for code, rules, kw in (
            (-2, R(), dict(tokens=i32(3))), (-2, R(), dict(tokens=cuda(4))), (-2, R(), dict(adjusted=cuda(4, 99))),
            (-1, R(), dict(tokens=i32(4, device=1))), (-2, R(), dict(adjusted=cuda(4, 100, dtype=torch.float16))),
            (-2, R(history=i32(4, 9)), {}), (-2, R(history=i32(3, 9), lengths=i32(4)), {}),
            (-2, R(history=i32(4, 9), lengths=i32(3)), {}), (-2, R(history=cuda(4, 9), lengths=i32(4)), {}),
            (-2, R(**history, recent=-1), {}), (-2, R(**history, penalties=cuda(2, 3)), {}), (-2, R(**history, penalties=cuda(4, 2)), {}),
            (-1, R(bias=cuda(4, 2)), {}), (-1, R(bias_tokens=i32(4, 2)), {}), (-2, R(bias=cuda(4, 2), bias_tokens=i32(4, 3)), {}),
            (-2, R(bias=cuda(3, 2), bias_tokens=i32(3, 2)), {}), (-2, R(bias=cuda(4, 2), bias_tokens=cuda(4, 2)), {}),
            (-2, R(allowed=i32(4, 3)), {}), (-2, R(allowed=i32(2, 4)), {}), (-2, R(allowed=cuda(4, 4)), {})):
        refused(code, lambda: focr_hip.select_tokens(x, 4, 100, rules, ctx=CTX, **({"tokens": to} | kw)))
    refused(-2, lambda: focr_hip.select_tokens(x, 4, 99, ctx=CTX, tokens=to))
    refused(-2, lambda: focr_hip.select_tokens(cuda(4, 100, contiguous=False), 4, 100, ctx=CTX, tokens=to))
