"""4-bit products of rows that hold infinities or NaNs: which outputs are infinite and
which NaN, that the other rows do not change, and that such a row does not hold the
others up."""
import numpy as np
import pytest

import gen
from gpu_util import F32, assert_bitwise, host, to_dev

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fh():
    import focr_hip

    return focr_hip


def matrix(fh, n, k, group, seed, columns=()):
    rng = np.random.Generator(np.random.PCG64(seed))
    codes = rng.integers(-8, 8, size=(n, k)).astype(np.int8)
    codes[:, columns] = 0
    scales = rng.uniform(1e-3, 9e-3, size=(n, -(-k // group))).astype(F32)
    vals = rng.standard_normal((n, len(columns))).astype(F32)
    lin = fh.QuantLinear(4, codes, scales, group, exc_cols=list(columns), exc_vals=vals)
    return lin, codes


def classes(x, codes):
    """A row's sums: NaN, or infinities of a sign (x holds some)."""
    with np.errstate(invalid="ignore"):
        if np.isnan(x).any():
            return np.full(len(codes), np.nan)
        return (x[np.isinf(x)] * codes[:, np.isinf(x)].astype(np.float64)).sum(axis=1)


SIZES = [(40, 129, 128), (768, 2304, 64), (5003, 1111, 32), (16384, 300, 64), (300, 9000, 64), (20000, 5000, 64)]


@pytest.mark.parametrize("epilogue", ["STORE", "ADD", "GLU"])
@pytest.mark.parametrize("rows", [3, 8])
@pytest.mark.parametrize("n,k,group", SIZES)
def test_classes_and_the_other_rows(fh, n, k, group, rows, epilogue):
    n -= n % 2
    lin, codes = matrix(fh, n, k, group, n + k)
    codes = codes.copy()
    wide = n // 2 if epilogue == "GLU" else n
    epi = fh.Epilogue[epilogue]
    base = gen.normal((rows, wide), 1.0, 3)
    x = gen.normal((rows, k), 1.0, 5)
    scale = np.abs(gen.normal((rows,), 1.0, 7)) + F32(0.5)
    call = lambda a: host(lin.linear_ex(to_dev(a), rows, row_scale=to_dev(scale), epilogue=epi, out=to_dev(base)))  # noqa: E731
    plain = call(x)
    for marked in ([(0, [k - 1], [np.inf])], [(1, [0, k // 2, k - 1], [np.inf, -np.inf, -np.inf]), (2, [k // 3], [np.nan])],
                   [(r, list(range(k)), [np.nan] * k) for r in range(rows)], [(2, [70, 71], [-np.inf, -np.inf])]):
        y = x.copy()
        for r, cols, values in marked:
            y[r, cols] = values
        got = call(y)
        bad = [r for r, _, _ in marked]
        keep = [r for r in range(rows) if r not in bad]
        assert_bitwise(got[keep], plain[keep], "the other rows")
        for r in bad:
            want = classes(y[r].astype(np.float64), codes)
            if epilogue == "GLU":
                with np.errstate(invalid="ignore"):
                    gate = np.where(want[0::2] > 0, want[0::2], np.where(np.isnan(want[0::2]), np.nan, 0.0))
                    want = gate * gate * want[1::2]
                # Which of the gate's NaNs a maximum with zero passes on is not asked here.
                fine = ~np.isnan(want)
                assert np.array_equal(got[r][fine], want[fine])
            else:
                assert np.array_equal(got[r], want.astype(F32), equal_nan=True), f"row {r}"


@pytest.mark.parametrize("rows", [2, 7])
def test_norms_make_nan(fh, rows):
    lin, _ = matrix(fh, 500, 1000, 64, 11)
    x = gen.normal((rows, 1000), 1.0, 13)
    plain = host(lin.linear_ex(to_dev(x), rows, rms_norm=True))
    y = x.copy()
    y[1, 300] = np.inf
    got = host(lin.linear_ex(to_dev(y), rows, rms_norm=True))
    assert np.isnan(got[1]).all()
    keep = [r for r in range(rows) if r != 1]
    assert_bitwise(got[keep], plain[keep])


@pytest.mark.parametrize("k", [1, 2, 3])
def test_short_rows(fh, k):
    lin, codes = matrix(fh, 30, k, 64, 17)
    x = gen.normal((4, k), 1.0, 19)
    x[1, k - 1], x[2, 0] = np.inf, np.nan
    got = host(lin.linear(to_dev(x), 4))
    for r in (1, 2):
        assert np.array_equal(got[r], classes(x[r].astype(np.float64), codes).astype(F32), equal_nan=True)
    assert np.isfinite(got[[0, 3]]).all()


@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_a_marked_row_does_not_hold_the_others_up(fh, value):
    # One row of eight, all of it NaN, or one infinity: within five times the call without it.
    import torch

    lin, _ = matrix(fh, 4096, 8192, 64, 23)
    x = gen.normal((8, 8192), 1.0, 29)
    y = x.copy()
    y[3, slice(None) if np.isnan(value) else 4000] = value

    def fastest(a):
        a, out = to_dev(a), torch.zeros(8, 4096, device="cuda:0")
        best = np.inf
        for _ in range(6):
            begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            lin.linear_ex(a, 8, out=out)
            begin.record()
            for _ in range(10):
                lin.linear_ex(a, 8, out=out)
            end.record()
            end.synchronize()
            best = min(best, begin.elapsed_time(end))
        return best

    assert fastest(y) <= 5 * fastest(x)
