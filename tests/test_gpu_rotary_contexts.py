"""A `Rotary` of one context with a cache of another, on streams of their own: bitwise the same
row step of one context."""
import numpy as np
import pytest

import gen
from gpu_util import F32, assert_bitwise, host, to_dev
from test_gpu_rotary import int32, pages_of, table

pytestmark = pytest.mark.gpu
ROWS = [3, 1, 20]


@pytest.fixture(scope="module")
def fh():
    import focr_hip

    return focr_hip


def own_stream(fh, ctx):
    """The context on its own stream, and that stream as torch's. None of torch's pool, which gives a stream out
    again after 32 others: one may hold a capture that a test of refusals has invalidated."""
    import torch

    ctx.use_stream(None)
    return torch.cuda.ExternalStream(fh.lib().focr_ctx_stream(ctx.handle), device="cuda:0")


def step(kv, rope, qkv, q=None):
    return kv.qkv_rows(qkv, rope, int32([0, 16, 5]), row_start=int32(np.concatenate([[0], np.cumsum(ROWS)])), q=q)


def test_a_table_made_behind_queued_work(fh):
    # The frequencies are computed on torch's stream, behind other work, and the cache's context is on a
    # stream that does not wait for it.
    import torch

    total = sum(ROWS)
    f, p, x = table(2, 16, 3), gen.normal((total, 2), 50.0, 5), gen.normal((total, 32 * 64), 1.0, 7)
    alone = pages_of(fh, [0, 16, 5], ROWS, 16, 8, 8, 16, 11)
    want = host(step(alone, fh.Rotary(f).at(to_dev(p)), to_dev(x)))
    ctx = fh.Context(0)
    kv = pages_of(fh, [0, 16, 5], ROWS, 16, 8, 8, 16, 11, ctx)
    lens, row_start = int32([0, 16, 5]), int32(np.concatenate([[0], np.cumsum(ROWS)]))
    positions, qkv, given = to_dev(p), to_dev(x), to_dev(f)
    q = torch.zeros(total, 16, 64, device="cuda:0")
    torch.cuda.synchronize()
    stream = own_stream(fh, ctx)
    torch.cuda._sleep(100_000_000)
    rotary = fh.Rotary(given * 1.0)  # of the default context, on torch's stream
    with torch.cuda.stream(stream):
        kv.qkv_rows(qkv, rotary.at(positions), lens, row_start=row_start, q=q)
    stream.synchronize()
    assert_bitwise(host(q), want, "queries")
    torch.cuda.synchronize()
    ctx.use_stream(torch.cuda.current_stream())
    for i, n in enumerate((0, 16, 5)):
        one = [-1] * 3
        one[i] = n
        starts = int32([0] * (i + 1) + [ROWS[i]] * (3 - i))
        for a, b in zip(kv.dequantize(ROWS[i], int32(one), row_start=starts), alone.dequantize(ROWS[i], int32(one), row_start=starts)):
            assert_bitwise(host(a), host(b), f"cache of sequence {i}")
    assert kv.refused() == alone.refused() == []


@pytest.mark.parametrize("owner", ["rotary", "cache"])
def test_a_rotary_that_is_dropped_while_its_table_is_read(fh, owner):
    # The call is queued behind other work on its stream when the rotary goes; torch's stream gives the
    # table's memory to other tensors at once.
    import torch

    total = sum(ROWS)
    f, p, x = table(2, 16, 3), gen.normal((total, 2), 50.0, 5), gen.normal((total, 32 * 64), 1.0, 7)
    alone = pages_of(fh, [0, 16, 5], ROWS, 16, 8, 8, 16, 11)
    want = host(step(alone, fh.Rotary(f).at(to_dev(p)), to_dev(x)))
    ctx = fh.Context(0)
    kv = pages_of(fh, [0, 16, 5], ROWS, 16, 8, 8, 16, 11, ctx)
    lens, row_start = int32([0, 16, 5]), int32(np.concatenate([[0], np.cumsum(ROWS)]))
    positions, qkv = to_dev(p), to_dev(x)
    q = torch.zeros(total, 16, 64, device="cuda:0")
    torch.cuda.synchronize()
    stream = own_stream(fh, ctx)
    rotary = fh.Rotary(f, ctx=ctx if owner == "rotary" else None)
    with torch.cuda.stream(stream):
        torch.cuda._sleep(100_000_000)
        kv.qkv_rows(qkv, rotary.at(positions), lens, row_start=row_start, q=q)
    del rotary
    other = [torch.full((2, 16, 32), 3.0, device="cuda:0") for _ in range(40)]
    torch.cuda.synchronize()
    assert_bitwise(host(q), want)
    assert len(other) == 40
    ctx.use_stream(torch.cuda.current_stream())
