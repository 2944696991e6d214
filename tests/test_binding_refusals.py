"""What the binding refuses before the library sees it, without a GPU: arrays
of fewer bytes than the call would read."""
import numpy as np
import pytest

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
