"""4-bit matrices whose exception columns have inputs far above the others', as they
exist for: the other columns' products keep FP32's accuracy."""
import numpy as np
import pytest

import gen
from gpu_util import F32, host, to_dev

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24  # half a step of FP32


@pytest.fixture(scope="module")
def fh():
    import focr_hip

    return focr_hip


def expected(x, w, columns, vals):
    """x w^T in 64 bits with the exceptions' products, and how far FP32's may be from it.

    The other inputs are off by 2^-22 of the largest other one of their block of 128, 256,
    384 or 512 columns; their sums round once for every 32 columns, for every block and
    a few times where bytes and waves meet. The exceptions are added one by one: a rounding
    each, and one of the whole."""
    rows, k = x.shape
    rest = x.copy()
    rest[:, columns] = 0
    big = np.zeros_like(x)
    for wide in (128, 256, 384, 512):
        most = np.abs(np.pad(rest, ((0, 0), (0, -k % wide)))).reshape(rows, -1, wide).max(axis=2)
        big = np.maximum(big, np.repeat(most, wide, axis=1)[:, :k])
    size = 1.02 * big @ np.abs(w).T
    bound = size * (4 * EPS + (1.25 * -(-k // 32) + 16) * EPS)
    outlying = np.abs(x[:, columns]) @ np.abs(vals.astype(np.float64)).T
    bound += (size + outlying) * (len(columns) + 2) * EPS
    return rest @ w.T + x[:, columns] @ vals.astype(np.float64).T, bound


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("large", [300.0, 1e4])
@pytest.mark.parametrize("n,k,group,columns", [(50, 768, 64, [0, 5, 700]), (33, 1111, 32, [3, 511, 512, 1108, 1110]), (64, 130, 128, [129]),
                                               (48, 6000, 64, [2, 3, 64, 5999]), (5003, 400, 32, [0, 255, 399])])
def test_large_inputs_of_exception_columns(fh, n, k, group, columns, large, norm):
    rng = np.random.Generator(np.random.PCG64(n + k))
    codes = rng.integers(-8, 8, size=(n, k)).astype(np.int8)
    codes[:, columns] = 0
    scales = rng.uniform(1e-3, 9e-3, size=(n, -(-k // group))).astype(F32)
    vals = (rng.standard_normal((n, len(columns))) * 1e-6).astype(F32)
    vals[::2] = 0
    lin = fh.QuantLinear(4, codes, scales, group, exc_cols=columns, exc_vals=vals)
    w = codes.astype(np.float64) * np.repeat(scales.astype(np.float64), group, axis=1)[:, :k]
    for rows in (1, 5, 8):
        x = gen.normal((rows, k), 1.0, rows + k)
        x[:, columns] *= F32(large)
        a, relative = x.astype(np.float64), 0.0
        if norm:
            # The factor's own error: a sum of squares rounds once for every 64 columns, its root and the rest a few times.
            a = a / np.sqrt((a * a).mean(axis=1, keepdims=True) + 2.0 ** -23)
            relative = (k / 64 + 16) * EPS
        want, bound = expected(a, w, columns, vals)
        got = host(lin.linear_ex(to_dev(x), rows, rms_norm=norm)).astype(np.float64)
        over = np.abs(got - want) / (bound + relative * np.abs(want))
        assert (over <= 1).all(), f"rows {rows}: {over.max()} times what is allowed"


@pytest.mark.parametrize("rows", [2, 8])
def test_exceptions_that_are_not_finite(fh, rows):
    # A marked row, whatever column its infinity stands in; the other rows keep their values.
    n, k, columns = 40, 3000, [7, 2999]
    rng = np.random.Generator(np.random.PCG64(5))
    codes = rng.integers(-8, 8, size=(n, k)).astype(np.int8)
    codes[:, columns] = 0
    scales = rng.uniform(1e-3, 9e-3, size=(n, -(-k // 64))).astype(F32)
    vals = rng.standard_normal((n, 2)).astype(F32)
    lin = fh.QuantLinear(4, codes, scales, 64, exc_cols=columns, exc_vals=vals)
    x = gen.normal((rows, k), 1.0, 3)
    x[0, 2999] = np.inf
    got = host(lin.linear(to_dev(x), rows))
    assert np.isnan(got[0]).all()  # infinity times a code of zero
    want, bound = expected(x[1:].astype(np.float64), codes * np.repeat(scales.astype(np.float64), 64, axis=1)[:, :k], columns, vals)
    assert (np.abs(got[1:] - want) <= bound).all()
