"""Attention over a shared prefix where rows are claimed twice and the prefix lacks a page: the
sequence that has the rows is named, as are those refused for claiming them."""
import numpy as np
import pytest

import gen
from gpu_util import assert_bitwise, host, to_dev
from test_gpu_pages import int32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fh():
    import focr_hip

    return focr_hip


# row_start of a batch; sequences that are accepted, and all that are refused once the prefix lacks a page.
@pytest.mark.parametrize("row_start,accepted,refused", [
    ([0, 4, 0, 4], [0], [0, 1, 2]),  # 1 ends before it begins, 2 claims all rows of 0
    ([0, 4, 2, 6, 0, 8], [0], [0, 1, 2, 3, 4]),  # 2 the last rows of 0, 4 all of 0 and more
    ([0, 1, 0, 1, 5], [0, 3], [0, 1, 2, 3]),  # 3 has rows of its own
])
@pytest.mark.parametrize("fill", [0, 80])  # rows of other sequences behind, so that waves take the tiles
@pytest.mark.parametrize("page", [16, 64])
def test_rows_claimed_twice_over_a_missing_page(fh, row_start, accepted, refused, fill, page):
    import torch

    shared, heads, group = 2 * page, 4, 2
    claims, last = len(row_start) - 1, row_start[-1]
    n, rows = claims + fill, last + fill
    row_start = row_start + list(range(last + 1, rows + 1))
    kv = fh.KvPages(2 + n, page, n + 1, 3, heads, heads // group, key_heads=heads // group)
    kv.map(n, 0, [0, 1])
    for i in range(n):
        kv.map(i, 2, [2 + i])
    k, v = (gen.normal((shared + 8 * n, heads // group, 64), 1.0, 3 + i) for i in range(2))
    kv.append(to_dev(k), to_dev(v), int32([shared] * n + [0]), row_start=int32(list(range(0, 8 * n + 1, 8)) + [8 * n + shared]))
    assert kv.refused() == []
    q = to_dev(gen.normal((rows, heads, 64), 1.0, 7))
    out = torch.full((rows, heads, 64), 5.0, device="cuda:0")
    call = lambda: kv.attention_shared(q, int32([shared] * n), shared + 8, shared, n, row_start=int32(row_start), out=out)  # noqa: E731
    others = list(range(claims, n))
    call()
    assert kv.refused() == [i for i in refused if i not in accepted]
    want = host(out)
    for i in accepted + others:
        assert np.isfinite(want[row_start[i]:row_start[i + 1]]).all(), i
    call()
    assert kv.refused() == [i for i in refused if i not in accepted]
    assert_bitwise(host(out), want)
    kv.map(n, 1, [-1])
    call()
    assert kv.refused() == refused + others
    got = host(out)
    for i in accepted + others:
        assert np.isnan(got[row_start[i]:row_start[i + 1]]).all(), i
