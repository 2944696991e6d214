"""4-bit matrices: decode GEMV, dequantization, prefill and refusals, against
64-bit sums."""
import numpy as np
import pytest

import gen
import oracle
from gpu_util import F32, assert_bitwise, host, to_dev

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24  # half a step of FP32


@pytest.fixture(scope="module")
def fh():
    import focr_hip

    return focr_hip


def matrix(n, k, group, seed, columns=()):
    rng = np.random.Generator(np.random.PCG64(seed))
    codes = rng.integers(-8, 8, size=(n, k)).astype(np.int8)
    scales = rng.uniform(1e-3, 9e-3, size=(n, -(-k // group))).astype(F32)
    vals = None
    if len(columns):
        codes[:, columns] = 0
        vals = rng.standard_normal((n, len(columns))).astype(F32)
    return codes, scales, vals


def weights64(codes, scales, group, columns=(), vals=None):
    w = codes.astype(np.float64) * np.repeat(scales.astype(np.float64), group, axis=1)[:, :codes.shape[1]]
    if len(columns):
        w[:, columns] = vals
    return w


def product(x, w):
    """x w^T in 64 bits, and how far FP32's may be from it. Inputs are integers of
    2^(e - 22), 2^e up to twice the largest of their block of 128, 256, 384 or 512
    columns, so off by 2^-22 of that; and sums of terms whose magnitudes add up to
    `size` (1.02 of it with the bytes' own magnitudes) round once for every 32
    columns, for every block, and a few times for the bytes' and waves' parts."""
    rows, k = x.shape
    big = np.zeros_like(x)
    for wide in (128, 256, 384, 512):
        pad = -k % wide
        most = np.abs(np.pad(x, ((0, 0), (0, pad)))).reshape(rows, -1, wide).max(axis=2)
        big = np.maximum(big, np.repeat(most, wide, axis=1)[:, :k])
    size = 1.02 * big @ np.abs(w).T
    groups = -(-k // 32)
    return x @ w.T, size * (4 * EPS + (1.25 * groups + 16) * EPS)


def normed(x):
    """RMS-normalized rows, and the relative error of FP32's."""
    k = x.shape[1]
    y = x / np.sqrt((x * x).mean(axis=1, keepdims=True) + 2.0 ** -23)
    return y, (k / 64 + 16) * EPS


def glu(y, err):
    g, u = np.maximum(y[:, 0::2], 0.0), y[:, 1::2]
    eg, eu = err[:, 0::2], err[:, 1::2]
    out = g * g * u
    bound = (g + eg) ** 2 * (np.abs(u) + eu) - g * g * np.abs(u)
    return out, bound + 3 * EPS * np.abs(out)


def check(got, want, bound, label=""):
    got = got.astype(np.float64)
    assert got.shape == want.shape, label
    over = np.abs(got - want) - bound - 1e-40
    assert (over <= 0).all(), f"{label}: off by {np.abs(got - want).max()} where {bound.max()} is allowed"


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k", [(1, 1), (3, 31), (37, 64), (16, 127), (40, 129), (33, 520), (48, 768), (5003, 1111),
                                 (2048, 768), (768, 2304), (9000, 200), (40000, 96)])
def test_decode_against_64_bits(fh, n, k, group):
    codes, scales, _ = matrix(n, k, group, 7 * n + k)
    lin = fh.QuantLinear.from_parts(n, k, group, codes, scales, bits=4)
    assert lin.bits() == 4
    w = weights64(codes, scales, group)
    for rows in (1, 2, 3, 4, 5, 6, 7, 8) if n < 3000 else (1, 5, 8):
        x = gen.values(rows * k, rows).reshape(rows, k) * F32(3.0)
        got = host(lin.linear(to_dev(x), rows))
        check(got, *product(x.astype(np.float64), w), f"n {n} k {k} group {group} rows {rows}")


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k", [(20, 20000), (300, 8200), (1000, 4100), (9000, 2304), (9000, 4100), (33000, 2200)])
def test_decode_of_large_calls(fh, n, k, group):
    # Rows written as bytes by a kernel of their own, and passed through LDS in turns.
    codes, scales, _ = matrix(n, k, group, n + k)
    lin = fh.QuantLinear.from_parts(n, k, group, codes, scales, bits=4)
    w = weights64(codes, scales, group)
    for rows in (1, 5, 8) if k > 8192 else (5, 8):
        x = gen.normal((rows, k), 2.0, rows)
        x[:, k // 3] *= 50.0
        got = host(lin.linear(to_dev(x), rows))
        check(got, *product(x.astype(np.float64), w), f"n {n} k {k} group {group} rows {rows}")


@pytest.mark.parametrize("n,k,group", [(16400, 3300, 32), (16400, 3300, 64), (16400, 3300, 128), (32768, 3300, 64)])
def test_decode_of_large_calls_with_many_channels(fh, n, k, group):
    # One wave a tile, in workgroups of six tiles and of eight.
    codes, scales, _ = matrix(n, k, group, n + k)
    lin = fh.QuantLinear.from_parts(n, k, group, codes, scales, bits=4)
    x = gen.normal((5, k), 2.0, 5)
    x[3, k // 3] = 40.0
    want, bound = product(x.astype(np.float64), weights64(codes, scales, group))
    check(host(lin.linear(to_dev(x), 5)), want, bound, f"n {n} k {k} group {group}")
    h = gen.normal((5, n), 1.0, 6)
    out = to_dev(h)
    lin.linear_ex(to_dev(x), 5, epilogue=fh.Epilogue.ADD, out=out)
    check(host(out), h + want, bound + EPS * (np.abs(h + want) + bound), f"ADD n {n} k {k} group {group}")


@pytest.mark.parametrize("n,k,group", [(64, 96, 32), (2048, 768, 64), (1030, 1300, 128), (4608, 768, 64), (70, 4500, 64)])
@pytest.mark.parametrize("rows", [1, 4, 5, 8])
def test_decode_with_its_neighbours(fh, n, k, group, rows):
    codes, scales, _ = matrix(n, k, group, n + k)
    lin = fh.QuantLinear.from_parts(n, k, group, codes, scales, bits=4)
    w = weights64(codes, scales, group)
    x = gen.values(rows * k, 3).reshape(rows, k)
    xd = to_dev(x)
    scale = gen.uniform(rows, 0.5, 1.5, 9).astype(F32)
    for name in ("plain", "row scale", "rms"):
        if name == "rms":
            a, rel = normed(x.astype(np.float64))
            kw = {"rms_norm": True}
        elif name == "row scale":
            a, rel = x.astype(np.float64) * scale[:, None].astype(np.float64), 0.0
            kw = {"row_scale": to_dev(scale)}
        else:
            a, rel, kw = x.astype(np.float64), 0.0, {}
        y, bound = product(a, w)
        bound = bound + (rel + EPS) * (np.abs(a) @ np.abs(w).T)
        check(host(lin.linear_ex(xd, rows, **kw)), y, bound, f"store {name}")
        check(host(lin.linear_ex(xd, rows, epilogue=fh.Epilogue.GLU, **kw)), *glu(y, bound), f"glu {name}")
        h = gen.values(rows * n, 5).reshape(rows, n)
        out = to_dev(h)
        lin.linear_ex(xd, rows, epilogue=fh.Epilogue.ADD, out=out, **kw)
        check(host(out), h + y, bound + 2 * EPS * np.abs(h + y), f"add {name}")
    y, bound = product(x.astype(np.float64), w)
    check(host(lin.linear_glu(xd, rows)), *glu(y, bound), "linear_glu")


@pytest.mark.parametrize("group,columns", [(64, [0]), (32, [3, 511, 767]), (128, [17, 18, 700])])
def test_exception_columns(fh, group, columns):
    n, k = 50, 768
    codes, scales, vals = matrix(n, k, group, 5, columns)
    lin = fh.QuantLinear(4, codes, scales, group, exc_cols=columns, exc_vals=vals)
    w = weights64(codes, scales, group, columns, vals)
    assert_bitwise(host(lin.dequantize()), w.astype(F32), "dequantize")  # fl(code * scale): one rounding
    for rows in (1, 5, 8):
        x = gen.values(rows * k, rows).reshape(rows, k)
        check(host(lin.linear(to_dev(x), rows)), *product(x.astype(np.float64), w), f"rows {rows}")


@pytest.mark.parametrize("n,k,group", [(1, 1, 64), (37, 129, 32), (48, 768, 64), (33, 300, 128)])
def test_dequantize_is_bit_exact(fh, n, k, group):
    codes, scales, _ = matrix(n, k, group, 11)
    lin = fh.QuantLinear.from_parts(n, k, group, codes, scales, bits=4)
    assert_bitwise(host(lin.dequantize()), weights64(codes, scales, group).astype(F32))


def test_inputs_of_every_magnitude(fh):
    # Rows and blocks of columns have exponents of their own.
    n, k, group = 64, 512, 64
    codes, scales, _ = matrix(n, k, group, 13)
    lin = fh.QuantLinear.from_parts(n, k, group, codes, scales, bits=4)
    w = weights64(codes, scales, group)
    x = gen.values(8 * k, 17).reshape(8, k).astype(np.float64)
    x[0] *= 1e30
    x[1] *= 1e-25
    x[2] *= np.repeat(10.0 ** np.arange(-12, 12, 3), 64)
    x[3] = 0.0
    x[4, 100] = 1e20
    x[5] *= 2.0 ** -100
    x = x.astype(F32)
    check(host(lin.linear(to_dev(x), 8)), *product(x.astype(np.float64), w))


@pytest.mark.parametrize("k", [200, 4200])
def test_rows_with_infinities_and_nans(fh, k):
    # Such a row is the FP32 sum of its products: an infinity times a code of zero
    # is NaN, and so are two infinities of different sign; the other rows keep their values.
    n, group = 300, 32
    codes, scales, _ = matrix(n, k, group, 19)
    codes[:, 7] = np.where(codes[:, 7] == 0, 1, codes[:, 7])
    codes[5, 7] = 0
    lin = fh.QuantLinear.from_parts(n, k, group, codes, scales, bits=4)
    w = weights64(codes, scales, group)
    x = gen.values(8 * k, 23).reshape(8, k)
    x[1, 7] = np.inf
    x[3, 7], x[3, 150] = -np.inf, np.inf
    x[6, 199] = np.nan
    got = host(lin.linear(to_dev(x), 8))
    with np.errstate(invalid="ignore"):
        want, bound = product(np.where(np.isfinite(x), x, 0).astype(np.float64), w)
        full = (x[:, None, :].astype(np.float64) * w[None]).sum(axis=2)
    for r in (0, 2, 4, 5, 7):
        check(got[r:r + 1], want[r:r + 1], bound[r:r + 1], f"row {r}")
    for r in (1, 3, 6):
        assert np.array_equal(np.isnan(got[r]), np.isnan(full[r])), r
        fine = ~np.isnan(full[r])
        assert np.array_equal(got[r][fine], full[r][fine].astype(F32)), r


def test_unaligned_rows_and_another_stream(fh):
    import torch

    n, k = 100, 66
    codes, scales, _ = matrix(n, k, 64, 29)
    ctx = fh.Context(0)
    lin = fh.QuantLinear.from_parts(n, k, 64, codes, scales, ctx=ctx, bits=4)
    w = weights64(codes, scales, 64)
    x = gen.values(3 * k + 1, 31)
    side = torch.cuda.Stream()
    xd = to_dev(x)
    side.wait_stream(torch.cuda.current_stream())
    ctx.use_stream(side)
    out = torch.empty(3 * n + 1, device="cuda:0")
    with torch.cuda.stream(side):
        lin.linear(xd[1:], 3, output=out[1:])
    side.synchronize()
    check(host(out)[1:].reshape(3, n), *product(x[1:].reshape(3, k).astype(np.float64), w))


def test_captured_steps_replay(fh):
    import torch

    n, k = 768, 2304
    codes, scales, _ = matrix(n, k, 64, 37)
    ctx = fh.Context(0)
    lin = fh.QuantLinear.from_parts(n, k, 64, codes, scales, ctx=ctx, bits=4)
    x = torch.zeros(5, k, device="cuda:0")
    out = torch.zeros(5, n, device="cuda:0")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ctx.use_stream(torch.cuda.current_stream())
        lin.linear_ex(x, 5, rms_norm=True, out=out)
    ctx.use_stream(torch.cuda.current_stream())
    for seed in range(4):
        x.copy_(to_dev(gen.values(5 * k, seed).reshape(5, k)))
        graph.replay()
        torch.cuda.synchronize()
        got = host(out)
        assert_bitwise(got, host(lin.linear_ex(x, 5, rms_norm=True)), f"replay {seed}")


def test_capture_needs_the_scratch_of_a_large_call(fh):
    import torch

    n, k = 64, 9000
    codes, scales, _ = matrix(n, k, 64, 71)
    ctx = fh.Context(0)
    lin = fh.QuantLinear.from_parts(n, k, 64, codes, scales, ctx=ctx, bits=4)
    x = torch.zeros(3, k, device="cuda:0")
    out = torch.zeros(3, n, device="cuda:0")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ctx.use_stream(torch.cuda.current_stream())
        with pytest.raises(fh.FocrError) as e:
            lin.linear(x, 3, output=out)
        out.add_(1.0)
    ctx.use_stream(torch.cuda.current_stream())
    assert e.value.code == -3
    lin.linear(x, 3, output=out)  # uncaptured: the scratch grows
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ctx.use_stream(torch.cuda.current_stream())
        lin.linear(x, 3, output=out)
    ctx.use_stream(torch.cuda.current_stream())
    for seed in range(3):
        x.copy_(to_dev(gen.normal((3, k), 1.0, seed)))
        graph.replay()
        torch.cuda.synchronize()
        got = host(out)
        assert_bitwise(got, host(lin.linear(x, 3)), f"replay {seed}")


@pytest.mark.parametrize("rows", [9, 40, 200])
@pytest.mark.parametrize("epilogue", ["STORE", "GLU", "ADD"])
def test_prefill_is_the_8_bit_matrixs(fh, rows, epilogue):
    # The codes as an 8-bit matrix: the same prefill kernels, bit for bit.
    n, k = 128, 192
    codes, scales, _ = matrix(n, k, 64, 41)
    four = fh.QuantLinear.from_parts(n, k, 64, codes, scales, bits=4)
    eight = fh.QuantLinear.from_parts(n, k, 64, codes, scales)
    x = to_dev(gen.values(rows * k, 43).reshape(rows, k))
    rs = to_dev(gen.uniform(rows, 0.5, 1.5, 47).astype(F32))
    epi = fh.Epilogue[epilogue]
    wide = n // 2 if epilogue == "GLU" else n
    for kernel in (fh.PrefillProjection.F32_MFMA, fh.PrefillProjection.F32_CHAIN, fh.PrefillProjection.I16):
        h = gen.values(rows * wide, 53).reshape(rows, wide)
        a, b = to_dev(h), to_dev(h)
        four.prefill(x, rows, row_scale=rs, epilogue=epi, out=a, kernel=kernel)
        eight.prefill(x, rows, row_scale=rs, epilogue=epi, out=b, kernel=kernel)
        assert_bitwise(host(a), host(b), f"{kernel.name} {epilogue} rows {rows}")


def test_prefill_of_odd_sizes(fh):
    n, k, rows = 37, 100, 11
    codes, scales, vals = matrix(n, k, 32, 59, [2, 99])
    four = fh.QuantLinear(4, codes, scales, 32, exc_cols=[2, 99], exc_vals=vals)
    eight = fh.QuantLinear(8, codes, scales, 32, exc_cols=[2, 99], exc_vals=vals)
    x = to_dev(gen.values(rows * k, 61).reshape(rows, k))
    for kernel in (fh.PrefillProjection.F32_MFMA, fh.PrefillProjection.F32_CHAIN):
        assert_bitwise(host(four.prefill(x, rows, kernel=kernel)), host(eight.prefill(x, rows, kernel=kernel)))
    with pytest.raises(fh.FocrError) as e:
        four.prefill(x, rows, kernel=fh.PrefillProjection.I16)
    assert e.value.code == -3
    with pytest.raises(fh.FocrError) as e:
        four.prefill(x, rows, kernel=fh.PrefillProjection.F32_SPLIT)
    assert e.value.code == -3


def test_refusals(fh):
    n, k = 20, 70
    codes, scales, _ = matrix(n, k, 64, 67)
    bad = codes.copy()
    bad[3, 69] = 8
    with pytest.raises(fh.FocrError) as e:
        fh.QuantLinear.from_parts(n, k, 64, bad, scales, bits=4)
    assert e.value.code == -5 and "[-8,7]" in str(e.value)
    bad[3, 69] = -9
    with pytest.raises(fh.FocrError):
        fh.QuantLinear.from_parts(n, k, 64, bad, scales, bits=4)
    for value in (np.nan, np.inf, -1.0, 2.0 ** 97):
        s = scales.copy()
        s[19, 1] = value
        with pytest.raises(fh.FocrError) as e:
            fh.QuantLinear.from_parts(n, k, 64, codes, s, bits=4)
        assert e.value.code == -5
    s = scales.copy()
    s[19, 1] = 0.0
    one = codes.copy()
    one[19, 64:] = 0
    one[19, 66] = 1
    with pytest.raises(fh.FocrError) as e:
        fh.QuantLinear.from_parts(n, k, 64, one, s, bits=4)
    assert e.value.code == -5 and "zero-scale" in str(e.value)
    one[19, 66] = 0
    fh.QuantLinear.from_parts(n, k, 64, one, s, bits=4)
    with pytest.raises(fh.FocrError) as e:
        fh.QuantLinear.from_parts(n, k, 16, codes, scales, bits=4)
    assert e.value.code == -2
    with pytest.raises(fh.FocrError):
        fh.QuantLinear.from_parts(n, k, 64, codes.astype(np.int16), scales, bits=4)
    with pytest.raises(fh.FocrError):
        fh.QuantLinear.from_parts(n, k, 64, codes, scales, bits=5)
    lin = fh.QuantLinear.from_parts(n, k, 64, codes, scales, bits=4)
    x = to_dev(np.zeros((9, k), F32))
    with pytest.raises(fh.FocrError) as e:
        lin.linear(x, 9)
    assert e.value.code == -2


def test_channels_past_31_bits_are_refused(fh):
    # Refused by its sizes alone, before any code is read.
    import ctypes

    codes, scales, out = np.zeros(1, np.int8), np.zeros(1, np.float32), ctypes.c_void_p()
    ptr = lambda a: a.ctypes.data_as(ctypes.c_void_p)  # noqa: E731
    rc = fh.lib().focr_linear_upload(fh.default_context().handle, 4, 2 ** 31 - 15, 1, 64, ptr(codes), ptr(scales), None,
                                     None, 0, ctypes.byref(out))
    assert rc == -2 and out.value is None
