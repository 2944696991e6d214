"""Batches whose sequences' rows overlap: what the append refuses, attention refuses,
and the other sequences' rows are as they are without it."""
import numpy as np
import pytest

import gen
from gpu_util import assert_bitwise, host, to_dev

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fh():
    import focr_hip

    return focr_hip


def int32(values):
    return to_dev(np.asarray(values, dtype=np.int32))


def plan(starts, lens, capacity, rows, max_len):
    """For each sequence its rows as (begin, end) if it is served, "refused" or "idle", and the rows that are NaN."""
    n = len(lens)
    what, reach, nan = [], 0, []
    for i in range(n):
        begin, end = starts[i], starts[i + 1]
        if lens[i] < 0:
            what.append("idle")
            continue
        fits = begin >= 0 and begin <= end <= rows and lens[i] + end - begin <= capacity
        served = fits and begin < end and begin >= reach and end - begin <= 8 and lens[i] + end - begin <= max_len
        if fits and begin < end:
            reach = max(reach, end)
        what.append((begin, end) if served else "idle" if fits and begin == end else "refused")
        if what[-1] == "refused" and begin >= 0 and end <= rows:
            nan += range(max(starts[:i + 1]), min(starts[i + 1:]))
    return what, nan


BATCHES = [([0, 4, 2, 4, 4], [20, 20, 20, 20]),  # 1 ends before it begins, 2 takes two of 0's rows
           ([0, 4, 2, 6, 8], [20, 20, 20, 20]),  # 2 takes two of 0's rows and two more; 3 is fine
           ([0, 4, 2, 4, 4], [-1, 20, 20, 20]),  # 0 takes no part: 2 is fine
           ([0, 4, 2, 4, 4], [500, 20, 20, 20]),  # 0 does not fit: its first two rows are its own, 2 is fine
           ([0, 9, 4, 7, 8], [20, 20, 20, 20]),  # 0 has nine rows
           ([0, 3, 3, 5, 8], [20, 20, 20, 20])]  # all fine


@pytest.mark.parametrize("starts,lens", BATCHES)
def test_plan_is_the_documents(starts, lens):
    what, nan = plan(starts, lens, 64, 10, 64)
    served = [w for w in what if isinstance(w, tuple)]
    taken = [r for b, e in served for r in range(b, e)]
    assert len(taken) == len(set(taken)) and not set(taken) & set(nan)


@pytest.mark.parametrize("max_len", [64, 4096])  # one part, and parts that a second kernel joins
@pytest.mark.parametrize("starts,lens", BATCHES)
@pytest.mark.parametrize("extra", [0, 300])  # sequences without rows before these
def test_overlapping_rows_are_refused_alone(fh, starts, lens, max_len, extra):
    import torch

    n, rows = 4 + extra, 10
    kv = fh.KvPages(n * 4, 16, n, max_len // 16, 16, 8)
    for i in range(extra, n):
        kv.map(i, 0, [4 * i + j for j in range(4)])
    held = int32([0] * n)
    k, v = gen.normal((4 * 40, 8, 64), 1.0, 3), gen.normal((4 * 40, 8, 64), 1.0, 5)
    kv.append(to_dev(k), to_dev(v), held, row_start=int32([0] * extra + [0, 40, 80, 120, 160]))
    assert kv.refused() == []
    if lens[0] == 500:
        lens = [max_len + 1] + lens[1:]
    q = to_dev(gen.normal((rows, 16, 64), 1.0, 7))
    what, nan = plan(starts, lens, max_len, rows, max_len)
    out = torch.full((rows, 16, 64), 5.0, device="cuda:0")
    kv.attention(q, int32([0] * extra + lens), max_len, row_start=int32([0] * extra + starts), out=out)
    refused = [extra + i for i, w in enumerate(what) if w == "refused"]
    assert kv.refused() == refused
    got = host(out)
    want = np.full((rows, 16, 64), 5.0, np.float32)
    want[nan] = np.nan
    for i, w in enumerate(what):
        if isinstance(w, tuple):
            # The sequence alone among idle ones.
            alone = [-1] * n
            alone[extra + i] = lens[i]
            begin, end = w
            one = kv.attention(q, int32(alone), max_len, row_start=int32([begin] * (extra + i + 1) + [end] * (4 - i)))
            want[begin:end] = host(one)[begin:end]
    assert_bitwise(got, want)
    assert kv.refused() == []
    # The append refuses the same ones but for too many rows.
    kv.append(to_dev(k[:rows]), to_dev(v[:rows]), int32([0] * extra + lens), row_start=int32([0] * extra + starts))
    assert kv.refused() == [r for r in refused if not (starts[r - extra + 1] - starts[r - extra] > 8)]
