"""What the binding refuses before the library sees it, without a GPU: arrays and
tensors of fewer bytes than the call would read or write."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import focr_hip

F32 = np.float32


def refused(code, call):
    with pytest.raises(focr_hip.FocrError) as e:
        call()
    assert e.value.code == code, str(e.value)


def codes(n=32, k=192, dtype=np.int8):
    return np.ones((n, k), dtype)


@pytest.mark.parametrize("bits", [4, 8, 16])
def test_scales_have_a_column_for_each_group(bits):
    c = codes(dtype=np.int16 if bits == 16 else np.int8)
    for shape in ((32, 3), (32, 2), (31, 6), (6, 32), (32,), ()):  # groups of 32: six
        refused(-2, lambda: focr_hip.Linear(bits, c, np.ones(shape, F32), 32))
    refused(-2, lambda: focr_hip.QuantLinear.from_parts(32, 192, 32, c, np.ones((32, 3), F32), bits=bits))
    refused(-2, lambda: focr_hip.Linear(bits, codes(32, 65, c.dtype), np.ones((32, 1), F32), 64))


@pytest.mark.parametrize("bits", [4, 8, 16])
def test_exceptions_have_a_weight_for_each_row(bits):
    c, s = codes(dtype=np.int16 if bits == 16 else np.int8), np.ones((32, 3), F32)
    c[:, [3, 7]] = 0
    for values in (np.ones((32, 1), F32), np.ones((31, 2), F32), np.ones((2, 32), F32), np.ones(2, F32), None):
        refused(-2, lambda: focr_hip.Linear(bits, c, s, 64, exc_cols=[3, 7], exc_vals=values))
    refused(-2, lambda: focr_hip.Linear(bits, c, s, 64, exc_cols=[[3, 7]], exc_vals=np.ones((32, 1), F32)))


@pytest.mark.parametrize("bits,bad", [(4, 260), (8, 256 + 5), (8, -129), (16, 1 << 16), (16, -32769)])
def test_codes_are_not_cut(bits, bad):
    c = codes(dtype=np.int64)
    c[5, 9] = bad
    refused(-5, lambda: focr_hip.Linear(bits, c, np.ones((32, 3), F32), 64))
    c = codes(dtype=np.float64)
    c[5, 9] = 1.5
    refused(-5, lambda: focr_hip.Linear(bits, c, np.ones((32, 3), F32), 64))


def test_other_matrices():
    refused(-1, lambda: focr_hip.Linear(5, codes(), np.ones((32, 3), F32), 64))
    refused(-1, lambda: focr_hip.Linear(8, codes()[0], np.ones((32, 3), F32), 64))


def cuda(*shape, dtype=torch.float32, device=0, contiguous=True):
    """Stands in for a CUDA tensor."""
    return SimpleNamespace(is_cuda=True, dtype=dtype, get_device=lambda: device, is_contiguous=lambda: contiguous,
                           data_ptr=lambda: 4096, numel=lambda: int(np.prod(shape)), shape=torch.Size(shape), device="meta")


def test_tensors_of_other_types_and_devices():
    dev = focr_hip._dev
    assert dev(cuda(4)) == 4096 and dev(cuda(4), 0) == 4096 and dev(None) is None
    for dtype in (torch.float16, torch.bfloat16, torch.float64, torch.int32):
        refused(-2, lambda: dev(cuda(4, dtype=dtype)))
    refused(-2, lambda: dev(cuda(4, contiguous=False)))
    refused(-1, lambda: dev(cuda(4, device=1), 0))
    refused(-1, lambda: dev(torch.zeros(4)))


def test_projections_refuse_what_they_would_read_or_write_past():
    lin = object.__new__(focr_hip.Linear)
    lin.ctx, lin.handle = SimpleNamespace(handle=None, device=0), None
    lin.out_dim, lin.in_dim = 32, 64
    x = cuda(2, 64)
    add = focr_hip.Epilogue.ADD
    for bad in (dict(dtype=torch.float16), dict(dtype=torch.bfloat16)):
        half = cuda(2, 64, **bad)
        for call in (lambda: lin.linear(half, 2, output=cuda(2, 32)), lambda: lin.linear(x, 2, output=cuda(2, 32, **bad)),
                     lambda: lin.linear_glu(half, 2, gated=cuda(2, 16)), lambda: lin.linear_glu(x, 2, gated=cuda(2, 16, **bad)),
                     lambda: lin.linear_ex(half, 2, out=cuda(2, 32)),
                     lambda: lin.linear_ex(x, 2, epilogue=add, out=cuda(2, 32, **bad)),
                     lambda: lin.linear_ex(x, 2, row_scale=cuda(2, **bad), out=cuda(2, 32)),
                     lambda: lin.prefill(half, 2, out=cuda(2, 32)),
                     lambda: lin.prefill(x, 2, epilogue=add, out=cuda(2, 32, **bad)),
                     lambda: focr_hip.row_scales(half, 64, out=cuda(2), ctx=lin.ctx)):
            refused(-2, call)
    for call in (lambda: lin.linear_glu(x, 2, gated=cuda(2, 15)), lambda: lin.linear_ex(x, 2, row_scale=cuda(1), out=cuda(2, 32)),
                 lambda: lin.prefill(x, 2, row_scale=cuda(1), out=cuda(2, 32)), lambda: lin.prefill(x, 2, out=cuda(1, 32))):
        refused(-2, call)
    for call in (lambda: lin.linear_ex(cuda(2, 64, device=1), 2, out=cuda(2, 32)),
                 lambda: lin.prefill(x, 2, epilogue=add, out=cuda(2, 32, device=1))):
        refused(-1, call)


def test_steps_refuse_other_hidden_states():
    layer, pages, ctx = object.__new__(focr_hip.DecoderLayer), object.__new__(focr_hip.KvPages), SimpleNamespace(handle=None, device=0)
    layer.ctx = pages.ctx = ctx
    layer.n_heads = pages.n_heads = 16
    layer.n_kv_heads = pages.n_kv_heads = 8
    layer.dim, pages.handle = 64, None
    pages._float, pages._int, pages._device = torch.float32, torch.int32, 0
    for code, h in ((-2, cuda(2, 64, dtype=torch.float16)), (-2, cuda(2, 64, dtype=torch.bfloat16)),
                    (-2, cuda(2, 64, contiguous=False)), (-1, cuda(2, 64, device=1)), (-2, cuda(2, 63))):
        refused(code, lambda: layer.decode_pages(h, None, pages, None, 16))
