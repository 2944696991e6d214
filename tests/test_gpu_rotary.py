"""Rotary positions with several axes: factors against 64 bits, and the paged row step that forms
them itself against factors and row step, bitwise."""
import numpy as np
import pytest

import gen
from gpu_util import F32, assert_bitwise, host, to_dev

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fh():
    import focr_hip

    return focr_hip


def int32(values):
    return to_dev(np.asarray(values, dtype=np.int32))


def factors64(positions, frequencies):
    """cos and sin in 64 bits of angles added axis by axis: products of FP32 are exact."""
    p, f = positions.astype(np.float64), frequencies.astype(np.float64)
    angle = p[:, 0, None, None] * f[0]
    for axis in range(1, p.shape[1]):
        angle = angle + p[:, axis, None, None] * f[axis]
    return np.stack([np.cos(angle), np.sin(angle)], axis=-1)


def check(got, want):
    """Half a step of FP32 from the 64-bit value, and what 64 bits are off: the reduced angle by two
    roundings of at most 2^-53, the sums by some ten of that, of values up to 1."""
    step = np.spacing(np.abs(want).astype(F32)).astype(np.float64)
    off = np.abs(got.astype(np.float64) - want)
    allowed = step / 2 + 16 * 2.0 ** -53
    assert (off <= allowed).all(), f"{(off / allowed).max()} times what is allowed at {np.unravel_index((off / allowed).argmax(), off.shape)}"


def table(axes, heads, seed, top=1.0):
    """Frequencies from `top` down to 2^-16 of it, of either sign, some of them zero."""
    rng = np.random.Generator(np.random.PCG64(seed))
    f = top * 2.0 ** -rng.uniform(0, 16, size=(axes, heads, 32)) * rng.choice([-1, 1], size=(axes, heads, 32))
    f[rng.random(f.shape) < 0.2] = 0
    return f.astype(F32)


@pytest.mark.parametrize("axes", [1, 2, 3, 4])
@pytest.mark.parametrize("rows,heads", [(1, 16), (2, 1), (5, 3), (2049, 16), (4500, 2), (70, 33)])
def test_factors(fh, axes, rows, heads):
    rng = np.random.Generator(np.random.PCG64(rows + axes))
    f = table(axes, heads, axes)
    p = rng.uniform(-50, 50, size=(rows, axes)).astype(F32)
    p[:, 0] = rng.integers(0, 200000, size=rows)
    p[::3, axes - 1] = 0
    rotary = fh.Rotary(f)
    want = factors64(p, f)
    got = host(rotary.factors(to_dev(p)))
    assert got.shape == (rows, heads, 32, 2)
    check(got, want)
    out = to_dev(np.full((rows + 2, heads, 32, 2), 7.0, F32))
    assert rotary.factors(to_dev(p), out=out[1:-1]).data_ptr() == out[1:].data_ptr()
    assert_bitwise(host(out)[1:-1], got)
    assert (host(out)[[0, -1]] == 7.0).all()  # rows before and behind stay


@pytest.mark.parametrize("top", [2.0 ** 20, 2.0 ** 33, 2.0 ** -40])
def test_angles_near_and_far(fh, top):
    # One axis, so that the angle is exact: up to 2^49, and down to 2^-70.
    f = table(1, 4, 3, top)
    p = np.array([[1.0], [-1.0], [0.0], [3.0], [65535.0], [0.001]], F32)
    check(host(fh.Rotary(f).factors(to_dev(p))), factors64(p, f))


def test_quarter_turns(fh):
    # Angles next to the multiples of pi / 4, where sine and cosine change places, near and far.
    rng = np.random.Generator(np.random.PCG64(5))
    k = np.concatenate([np.arange(-40, 41), rng.integers(-2 ** 22, 2 ** 22, size=200)])
    f = np.repeat((k * np.pi / 4).astype(F32).reshape(1, -1, 1), 32, axis=2)
    f *= (1 + (np.arange(32) - 16) * 2.0 ** -23).astype(F32)
    p = np.array([[1.0]], F32)
    check(host(fh.Rotary(f).factors(to_dev(p))), factors64(p, f))


def test_angles_that_are_none(fh):
    f = np.ones((2, 2, 32), F32)
    f[0] = 2.0
    p = np.array([[np.inf, 0], [0, np.nan], [2.0 ** 51, 0], [-2.0 ** 60, 1], [3e38, -3e38], [2.0 ** 47, 0]], F32)
    got = host(fh.Rotary(f).factors(to_dev(p)))
    assert np.isnan(got[:5]).all()
    check(got[5:], factors64(p[5:], f))


def test_tables_of_other_types(fh):
    import torch

    f, p = table(2, 4, 9), gen.normal((6, 2), 9.0, 11)
    want = host(fh.Rotary(f).factors(to_dev(p)))
    for other in (f.astype(np.float64), torch.from_numpy(f), to_dev(f), to_dev(f).permute(1, 0, 2).contiguous().permute(1, 0, 2)):
        assert_bitwise(host(fh.Rotary(other).factors(to_dev(p))), want)
    given = to_dev(f)
    rotary = fh.Rotary(given)
    given.zero_()  # the table is the operator's own
    assert_bitwise(host(rotary.factors(to_dev(p))), want)


def pages_of(fh, lens, rows, heads, kv_heads, key_heads, page, seed, ctx=None):
    counts = [max(1, -(-(n + r) // page)) for n, r in zip(lens, rows)]
    kv = fh.KvPages(sum(counts) + 2, page, len(lens), max(counts), heads, kv_heads, key_heads=key_heads, ctx=ctx)
    ids = np.random.Generator(np.random.PCG64(seed)).permutation(sum(counts) + 2)
    at = 0
    for i, n in enumerate(counts):
        kv.map(i, 0, ids[at:at + n])
        at += n
    return kv


@pytest.mark.parametrize("heads,kv_heads,key_heads", [(16, 8, 8), (16, 8, 16), (4, 4, 4), (6, 1, 1), (6, 3, 6)])
@pytest.mark.parametrize("axes", [1, 2, 3, 4])
def test_row_step_from_positions(fh, heads, kv_heads, key_heads, axes):
    # Short and long rows, behind whole and cut blocks, one idle sequence and one without rows.
    lens, rows = [0, 5, 16, 31, 40, 3, 7], [1, 3, 40, 1, 0, 200, 2]
    held = [n if i != 6 else -1 for i, n in enumerate(lens)]
    total = sum(rows)
    row_start = int32(np.concatenate([[0], np.cumsum(rows)]))
    kvs = [pages_of(fh, lens, rows, heads, kv_heads, key_heads, 16, 3) for _ in range(2)]
    k0, v0 = gen.normal((sum(lens), key_heads, 64), 1.0, 5), gen.normal((sum(lens), kv_heads, 64), 1.0, 7)
    for kv in kvs:
        kv.append(to_dev(k0), to_dev(v0), int32([0] * 7), row_start=int32(np.concatenate([[0], np.cumsum(lens)])))
    qkv = to_dev(gen.normal((total, (heads + 2 * kv_heads) * 64), 1.0, 11))
    p = gen.normal((total, axes), 30.0, 13)
    p[:, 0] = np.arange(total) + 70000
    positions, rotary = to_dev(p), fh.Rotary(table(axes, heads, 17))
    outs = [to_dev(np.full((total, heads, 64), 5.0, F32)) for _ in kvs]
    kvs[0].qkv_rows(qkv, rotary.at(positions), int32(held), row_start=row_start, q=outs[0])
    kvs[1].qkv_rows(qkv, rotary.factors(positions), int32(held), row_start=row_start, q=outs[1])
    assert_bitwise(host(outs[0]), host(outs[1]), "queries")
    assert (host(outs[0])[-2:] == 5.0).all() and (host(outs[0])[:-2] != 5.0).any(axis=2).all()
    after = [n + (r if h >= 0 else 0) for n, r, h in zip(lens, rows, held)]
    read = int32(np.concatenate([[0], np.cumsum(after)]))
    for a, b in zip(*(kv.dequantize(sum(after), int32([0] * 7), row_start=read) for kv in kvs)):
        assert_bitwise(host(a), host(b), "cache")
    assert kvs[0].refused() == kvs[1].refused() == []


def test_long_prompts_from_positions(fh):
    # The grid of long prompts.
    lens, rows = [9, 0], [1500, 1100]
    row_start = int32([0, 1500, 2600])
    qkv = to_dev(gen.normal((2600, 32 * 64), 1.0, 19))
    positions, rotary = to_dev(gen.normal((2600, 3), 40.0, 23)), fh.Rotary(table(3, 16, 29))
    got = []
    for rope in (rotary.at(positions), rotary.factors(positions)):
        kv = pages_of(fh, lens, rows, 16, 8, 16, 64, 31)
        q = kv.qkv_rows(qkv, rope, int32(lens), row_start=row_start)
        got.append([host(q)] + [host(t) for t in kv.dequantize(2600, int32(lens), row_start=row_start)])
    for a, b in zip(*got):
        assert_bitwise(a, b)


def test_captured_steps_read_their_positions(fh):
    # One graph of factors and row steps; positions and lengths are advanced by it.
    import torch

    ctx = fh.Context(0)
    n, steps = 5, 20
    lens, rows = [0, 15, 16, 3, 30], [steps] * 5
    kv, other = (pages_of(fh, lens, rows, 16, 8, 8, 16, 37, ctx) for _ in range(2))
    k0, v0 = gen.normal((sum(lens), 8, 64), 1.0, 41), gen.normal((sum(lens), 8, 64), 1.0, 43)
    for c in (kv, other):
        c.append(to_dev(k0), to_dev(v0), int32([0] * n), row_start=int32(np.concatenate([[0], np.cumsum(lens)])))
    rotary = fh.Rotary(table(2, 16, 47), ctx=ctx)
    positions = to_dev(np.stack([np.array(lens), np.zeros(n)], axis=1).astype(F32))
    at, qkv = int32(lens), torch.zeros(n, 32 * 64, device="cuda:0")
    q, factors = torch.zeros(n, 16, 64, device="cuda:0"), torch.zeros(n, 16, 32, 2, device="cuda:0")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ctx.use_stream(torch.cuda.current_stream())
        rotary.factors(positions, out=factors)
        kv.qkv_rows(qkv, rotary.at(positions), at, q=q)
        positions[:, 0].add_(1.0)
        at.add_(1)
    ctx.use_stream(torch.cuda.current_stream())
    for step in range(steps):
        qkv.copy_(to_dev(gen.normal((n, 32 * 64), 1.0, 53 + step)))
        graph.replay()
        torch.cuda.synchronize()
        p = to_dev(np.stack([np.array(lens) + step, np.zeros(n)], axis=1).astype(F32))
        want = rotary.factors(p)
        assert_bitwise(host(factors), host(want), f"factors of step {step}")
        assert_bitwise(host(q), host(other.qkv_rows(qkv, want, int32([x + step for x in lens]))), f"step {step}")
    assert kv.refused() == []


def test_another_stream(fh):
    import torch

    f, p = table(3, 16, 59), gen.normal((300, 3), 100.0, 61)
    want = host(fh.Rotary(f).factors(to_dev(p)))
    ctx, stream = fh.Context(0), torch.cuda.Stream()
    ctx.use_stream(stream)
    rotary = fh.Rotary(f, ctx=ctx)  # its table is made on torch's stream
    x = to_dev(p)
    out = torch.zeros(300, 16, 32, 2, device="cuda:0")
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        rotary.factors(x, out=out)
    stream.synchronize()
    assert_bitwise(host(out), want)


def test_refusals(fh):
    import torch

    def refused(code, call):
        with pytest.raises(fh.FocrError) as e:
            call()
        assert e.value.code == code, str(e.value)

    x = lambda *shape, **kw: torch.ones(*shape, device="cuda:0", **kw)  # noqa: E731
    for shape in ((5, 16, 32), (0, 16, 32), (2, 16, 31), (16, 32), (1, 0, 32)):
        if shape == (1, 0, 32):
            refused(-2, lambda: fh.Rotary(np.ones(shape, F32)).factors(x(1, 1)))
        else:
            refused(-2, lambda: fh.Rotary(np.ones(shape, F32)))
    rotary = fh.Rotary(np.ones((2, 16, 32), F32))
    refused(-2, lambda: rotary.factors(x(4, 3)))
    refused(-2, lambda: rotary.factors(x(8)))
    refused(-2, lambda: rotary.factors(x(4, 2, dtype=torch.float64)))
    refused(-2, lambda: rotary.factors(x(4, 4)[:, ::2]))
    refused(-1, lambda: rotary.factors(torch.ones(4, 2), out=x(4, 16, 32, 2)))
    refused(-2, lambda: rotary.factors(x(4, 2), out=x(3, 16, 32, 2)))
    refused(-1, lambda: rotary.factors(x(4, 2), out=x(4 * 1024 + 1)[1:]))  # not on 16 bytes
    assert rotary.factors(x(0, 2)).shape == (0, 16, 32, 2)
    kv = fh.KvPages(4, 16, 2, 2)
    lens = int32([0, 0])
    refused(-2, lambda: kv.qkv_rows(x(2, 32 * 64), rotary.at(x(3, 2)), lens))
    refused(-2, lambda: kv.qkv_rows(x(2, 32 * 64), fh.Rotary(np.ones((2, 8, 32), F32)).at(x(2, 2)), lens))
    refused(-2, lambda: kv.qkv_rows(x(2, 32 * 64), rotary.at(x(2, 2, dtype=torch.float16)), lens))
    refused(-2, lambda: rotary.at(x(2, 3)))
