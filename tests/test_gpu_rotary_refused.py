"""The paged row step from positions where sequences are refused, overlap, take no part or miss a
page: bitwise factors and then the row step, with the same sequences named."""
import numpy as np
import pytest

import gen
from gpu_util import F32, assert_bitwise, host, to_dev
from test_gpu_pages_overlap import BATCHES
from test_gpu_rotary import int32, table

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fh():
    import focr_hip

    return focr_hip


def both(fh, caches, heads, kv_heads, rows, lens, row_start, axes, label):
    """The step by positions and by factors; what they leave, and whom they name."""
    qkv = to_dev(gen.normal((rows, (heads + 2 * kv_heads) * 64), 1.0, 11))
    positions, rotary = to_dev(gen.normal((rows, axes), 300.0, 13)), fh.Rotary(table(axes, heads, 17))
    outs = [to_dev(np.full((rows + 2, heads, 64), 5.0, F32)) for _ in caches]
    for kv, rope, out in zip(caches, (rotary.at(positions), rotary.factors(positions)), outs):
        kv.qkv_rows(qkv, rope, int32(lens), row_start=row_start, q=out[1:-1])
    got, want = (host(t) for t in outs)
    assert_bitwise(got, want, f"{label}: queries")
    assert (got[[0, -1]] == 5.0).all()
    named = [kv.refused() for kv in caches]
    assert named[0] == named[1], label
    for i in range(len(lens)):
        # All of a sequence's positions; the other sequences take no part.
        alone, every = [-1] * len(lens), caches[0].seq_pages * caches[0].page_size
        alone[i] = 0
        starts = int32([0] * (i + 1) + [every] * (len(lens) - i))
        for a, b in zip(*(kv.dequantize(every, int32(alone), row_start=starts) for kv in caches)):
            assert_bitwise(host(a), host(b), f"{label}: sequence {i}")
    for kv in caches:
        kv.refused()  # sequences without all their pages, by reading back
    return named[0]


def caches_of(fh, n, pages, heads=16, kv_heads=8, page=16):
    out = []
    for _ in range(2):
        kv = fh.KvPages(n * pages, page, n, pages, heads, kv_heads, key_heads=kv_heads)
        for i in range(n):
            kv.map(i, 0, [pages * i + j for j in range(pages)])
        held = pages * page // 2 + 3
        k, v = (gen.normal((n * held, kv_heads, 64), 1.0, 3 + j) for j in range(2))
        kv.append(to_dev(k), to_dev(v), int32([0] * n), row_start=int32([held * i for i in range(n + 1)]))
        assert kv.refused() == []
        out.append(kv)
    return out


@pytest.mark.parametrize("starts_,lens", BATCHES)
@pytest.mark.parametrize("axes", [1, 3])
def test_overlapping_and_broken_batches(fh, starts_, lens, axes):
    # Rows that overlap, end before they begin, or leave the call; lengths past the pages.
    both(fh, caches_of(fh, 4, 4), 16, 8, 10, lens, int32(starts_), axes, str((starts_, lens)))


def test_refused_idle_and_without_a_page(fh):
    # 0 idle, 1 fine, 2 past its pages, 3 its first block's page missing, 4 the last's, 5 without rows, 6 fine.
    counts, lens = [2, 3, 20, 30, 40, 0, 5], [-1, 30, 60, 14, 20, 9, 31]
    caches = caches_of(fh, 7, 4)
    for kv in caches:
        kv.map(3, 0, [-1])
        kv.map(4, 3, [-1])
    starts_ = int32(np.concatenate([[0], np.cumsum(counts)]))
    named = both(fh, caches, 16, 8, sum(counts), lens, starts_, 2, "ragged")
    assert named == [2, 3, 4]


def test_single_rows_without_row_start(fh):
    lens = [5, -1, 64, 48, 0]
    caches = caches_of(fh, 5, 4)
    for kv in caches:
        kv.map(3, 3, [-1])
    assert both(fh, caches, 16, 8, 5, lens, None, 4, "single rows") == [2, 3]


def test_a_long_prompt_over_a_missing_page(fh):
    # The grid of long prompts.
    caches = caches_of(fh, 2, 20, page=64)
    for kv in caches:
        kv.map(0, 9, [-1])
    named = both(fh, caches, 16, 8, 1900, [100, 300], int32([0, 1000, 1900]), 3, "long")
    assert named == [0]
