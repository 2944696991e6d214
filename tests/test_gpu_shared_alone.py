"""Attention over a shared prefix where many short sequences have a wave for each part of their own
positions: several parts, positions that end with one, pages missing in a later one."""
import numpy as np
import pytest

from gpu_util import assert_bitwise, host
from test_gpu_shared import Batch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fh():
    import focr_hip

    return focr_hip


# More than 256 sequences and key heads together, at most four columns a sequence in the mean, and up to
# 1,024 own positions: parts of 512 (1,024 waves over 384 units: two each) and of 256 (over 264: three).
@pytest.mark.parametrize("n,key_heads,own,part", [(48, 8, 1000, 512), (48, 8, 1024, 512), (33, 8, 768, 256), (17, 16, 600, 256)])
@pytest.mark.parametrize("page", [16, 64, 128])
def test_parts_of_a_wave_each(fh, n, key_heads, own, part, page):
    shared = 128
    counts = [0 if i == 5 else 6 if i == 7 else 3 if i == 11 else 1 for i in range(n)]
    ends = {0: part, 1: part + 1, 2: part - 1, 3: 2 * part if 2 * part <= own else own, 4: 1, 6: own, 7: part + 3, 8: 16, 9: part + 16}
    owns = [ends[i] - counts[i] if i in ends else (own - counts[i]) * (7 * i % n) // n for i in range(n)]
    b = Batch(fh, shared, owns, counts, page, 16, 8, key_heads, seed=own + page + n)
    b.verify(host(b.shared_call(max_len=shared + own)))
    assert b.kv.refused() == []
    got = host(b.shared_call(max_len=shared + own))
    # A page behind the first part is missing for one sequence, another stands before the prefix's end.
    b.kv.map(6, (shared + part) // page, [-1])
    b.before[10] = shared - 1
    again = host(b.shared_call(max_len=shared + own))
    assert b.kv.refused() == [6, 10]
    first = np.concatenate([[0], np.cumsum(counts)])
    lost = np.zeros(len(got), bool)
    for i in (6, 10):
        lost[first[i]:first[i + 1]] = True
    assert np.isnan(again[lost]).all()
    assert_bitwise(again[~lost], got[~lost])


def test_others_that_take_no_part_change_nothing(fh):
    b, c = (Batch(fh, 64, [300] * 40, [1] * 40, 16, 16, 8, 8, seed=3) for _ in range(2))
    want = host(b.shared_call())
    c.before[20:] = [-1] * 20
    got = host(c.shared_call(max_len=max(b.totals)))
    assert_bitwise(got[:20], want[:20])
    assert b.kv.refused() == c.kv.refused() == []
