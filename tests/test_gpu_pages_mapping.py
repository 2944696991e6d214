"""Pages of a sequence mapped again: a block that is not full keeps its FP32 rows where
the page stays, and no longer than they are what the page holds."""
import numpy as np
import pytest

from gpu_util import assert_bitwise, host, to_dev
from test_gpu_pages import BLOCK, decoded, decoded_block, int32, rows_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fh():
    import focr_hip

    return focr_hip


def append(kv, seq, at, k, v):
    """Rows of sequence 0 or 1 of two, from position `at` on."""
    n = len(k)
    kv.append(to_dev(k), to_dev(v), int32([at, -1] if seq == 0 else [-1, at]), row_start=int32([0, n, n] if seq == 0 else [0, 0, n]))


def held(kv, seq, n):
    got = kv.dequantize(n, int32([0, -1] if seq == 0 else [-1, 0]), row_start=int32([0, n, n] if seq == 0 else [0, 0, n]))
    return [host(x) for x in got]


def rows(n, seed, scale=1.0):
    return rows_of([n], 8, seed, scale)[0], rows_of([n], 8, seed + 500, scale)[0]


@pytest.mark.parametrize("page,length", [(16, 5), (16, 21), (64, 21), (64, 70)])
def test_a_list_that_grows_is_sent_whole(fh, page, length):
    # Every call maps all pages so far again; the blocks are those of the rows, coded once.
    kv = fh.KvPages(40, page, 2, 20)
    k, v = rows(length + 30, 3)
    k[length:] *= np.float32(3.0)
    v[length:] *= np.float32(3.0)
    ids = list(range(30, 30 - (length + 30 + page - 1) // page, -1))
    at = 0
    for n in (length, 1, 2, 7, 20):
        kv.map(0, 0, ids[:(at + n + page - 1) // page])
        append(kv, 0, at, k[at:at + n], v[at:at + n])
        at += n
        for got, x in zip(held(kv, 0, at), (k, v)):
            assert_bitwise(got, decoded(x[:at]), f"after {at}")


def test_a_page_that_another_sequence_wrote_since(fh):
    # The table's entry is the same, the page's block is not: its codes are taken.
    kv = fh.KvPages(4, BLOCK, 2, 2)
    kv.map(0, 0, [2])
    append(kv, 0, 0, *rows(6, 5, 4.0))
    kv.map(1, 0, [2])
    other = rows(9, 7)
    append(kv, 1, 0, *other)
    kv.map(0, 0, [2])
    new = rows(3, 11, 2.0)
    append(kv, 0, 9, *new)
    for got, x, y in zip(held(kv, 0, 12), other, new):
        assert_bitwise(got, decoded_block(np.concatenate([decoded(x), y])))


def test_a_page_that_went_and_came_back(fh):
    kv = fh.KvPages(4, BLOCK, 2, 2)
    first, second, new = rows(6, 13), rows(6, 17, 4.0), rows(3, 19, 2.0)
    kv.map(0, 0, [2])
    append(kv, 0, 0, *first)
    kv.map(0, 0, [3])
    append(kv, 0, 0, *second)
    kv.map(0, 0, [2])
    append(kv, 0, 6, *new)
    for got, x, y in zip(held(kv, 0, 9), first, new):
        assert_bitwise(got, decoded_block(np.concatenate([decoded(x), y])))
    # And without a page in between.
    kv.map(0, 0, [-1])
    kv.map(0, 0, [2])
    before = held(kv, 0, 9)
    more = rows(2, 23, 5.0)
    append(kv, 0, 9, *more)
    for got, x, y in zip(held(kv, 0, 11), before, more):
        assert_bitwise(got, decoded_block(np.concatenate([x, y])))
