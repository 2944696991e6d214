"""Attention over the 8-bit cache of pages where its keys' weights and values are far
apart: as FP32 sums are, with no term for values that carry no weight."""
import numpy as np
import pytest

import gen
from gpu_util import F32, host, to_dev

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24  # half a step of FP32
HEADS = 2


@pytest.fixture(scope="module")
def fh():
    import focr_hip

    return focr_hip


def int32(values):
    return to_dev(np.asarray(values, dtype=np.int32))


def attention64(q, k, v, first):
    """64-bit attention of rows [n][heads][64] at positions first.., and how far FP32's may
    be from it.

    A score is off by the query's step (2^-22 of its largest element at most) times the key, and by
    a few roundings of itself and of its exponent; a weight by the exponential of twice that
    (its own and the maximum's). A weighted value passes a rounding, of up to a whole step
    where a matrix instruction cuts, for each of the terms that are added to it, of which a
    wave's run here has 1,024 at most; and some 100 where runs and parts meet, in the weight
    and in the division. All of these are relative to the sum of the magnitudes."""
    n, heads, _ = q.shape
    out, bound = np.empty(q.shape), np.empty(q.shape)
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    for h in range(heads):
        for r in range(n):
            seen = first + r + 1
            kh, vh = k[:seen, h], v[:seen, h]
            s = kh @ q[r, h] / 8.0
            w = np.exp(s - s.max())
            w /= w.sum()
            out[r, h] = w @ vh
            off = 4 * EPS * np.abs(q[r, h]).max() * np.abs(kh).sum(axis=1).max() / 8 + EPS * (8 * np.abs(s).max() + 16)
            bound[r, h] = w @ np.abs(vh) * (2.2 * off + EPS * (2 * min(seen, 1024) + 112)) + 1e-40
    return out, bound


def attend(fh, k, v, q, first, page=64):
    total = len(k)
    count = -(-total // page)
    kv = fh.KvPages(count, page, 1, count, HEADS, HEADS)
    kv.map(0, 0, list(range(count))[::-1])
    kv.append(to_dev(k.astype(F32)), to_dev(v.astype(F32)), int32([0]), row_start=int32([0, total]))
    gk, gv = (host(x) for x in kv.dequantize(total, int32([0]), row_start=int32([0, total])))
    got = host(kv.attention(to_dev(q), int32([first]), total, row_start=int32([0, len(q)])))
    want, bound = attention64(q, gk, gv, first)
    off = np.abs(got.astype(np.float64) - want)
    assert kv.refused() == [] and np.isfinite(got).all()
    assert (off <= bound).all(), f"{np.max(off / bound)} times what is allowed, off by {off.max()} of {np.abs(want).max()}"


def inputs(total, seed):
    return gen.normal((total, HEADS, 64), 1.0, seed), gen.normal((total, HEADS, 64), 1.0, seed + 1), gen.normal((1, HEADS, 64), 1.0, seed + 2)


def key_for(q, score):
    """Keys [heads][64] whose scores with q [1][heads][64] are `score`."""
    return q[0] * (8.0 * score / (q[0] * q[0]).sum(axis=1, keepdims=True))


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("total", [40, 1100])
@pytest.mark.parametrize("ratio", [1e6, 1e12, 1e30])
def test_large_values_without_weight(fh, total, ratio, page):
    # A block of large values at scores 100 below the others', as early in the run as not.
    for at in (0, total // 2 // 16 * 16):
        k, v, q = inputs(total, 7 + at)
        k[at:at + 16] = key_for(q, -100.0)
        v[at:at + 16] *= F32(ratio)
        attend(fh, k, v, q, total - 1, page)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("total", [40, 1100])
@pytest.mark.parametrize("gap", [14.0, 20.0, 40.0])
def test_a_first_key_that_takes_the_weight_and_has_no_value(fh, total, gap, page):
    # Weights of e^-gap carry the whole result: half the dims' for a value of zeros there.
    k, v, q = inputs(total, 31)
    k[3] = key_for(q, gap)
    v[3] = 0
    attend(fh, k, v, q, total - 1, page)
    v[3, :, ::2] = 50.0
    attend(fh, k, v, q, total - 1, page)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("ratio", [1e6, 1e30])
def test_large_values_behind_a_row(fh, ratio, page):
    # The first row does not see the block of the others.
    for base in (32, 1024):
        k, v, _ = inputs(base + 3, 43)
        v[base:] *= F32(ratio)
        attend(fh, k, v, gen.normal((4, HEADS, 64), 1.0, 47), base - 1, page)


@pytest.mark.parametrize("scale", [1e-34, 1e-20, 1e20, 1e35])
def test_values_of_one_small_or_large_magnitude(fh, scale):
    k, v, q = inputs(300, 53)
    attend(fh, k, v * F32(scale), q, 299)


@pytest.mark.parametrize("total", [40, 1100])
@pytest.mark.parametrize("large", [1e4, 3e5])
def test_a_large_query_element_that_meets_no_key(fh, total, large):
    # Scores come from elements far below the largest one. They are off by 2^-30 of that (half a
    # step of an integer that twice the largest bounds by 2^30) times the key, and by the roundings
    # of their own terms' sum and of the exponent.
    k, v, q = inputs(total, 59)
    k[:, :, 5] = 0
    q[:, :, 5] = large
    kv = fh.KvPages(-(-total // 64), 64, 1, -(-total // 64), HEADS, HEADS)
    kv.map(0, 0, list(range(-(-total // 64))))
    kv.append(to_dev(k), to_dev(v), int32([0]), row_start=int32([0, total]))
    gk, gv = (host(x).astype(np.float64) for x in kv.dequantize(total, int32([0]), row_start=int32([0, total])))
    got = host(kv.attention(to_dev(q), int32([total - 1]), total)).astype(np.float64)
    for h in range(HEADS):
        s = gk[:, h] @ q[0, h].astype(np.float64) / 8.0
        w = np.exp(s - s.max())
        w /= w.sum()
        step = 2.0 ** -30 * large * np.abs(gk[:, h]).sum(axis=1).max() / 8
        off = step + EPS * (6 * (np.abs(gk[:, h]) @ np.abs(q[0, h])).max() / 8 + 8 * np.abs(s).max() + 16)
        bound = w @ np.abs(gv[:, h]) * (2.2 * off + EPS * (2 * min(total, 1024) + 112))
        over = np.abs(got[0, h] - w @ gv[:, h]) / bound
        assert (over <= 1).all(), f"head {h}: {over.max()} times what is allowed"


@pytest.mark.parametrize("total", [130, 1100])
def test_value_blocks_far_apart_in_scale(fh, total):
    # Scales 2^133 apart: the smaller ones' products stay whole, before the large block and behind it.
    for at in (0, total // 2 // 16 * 16):
        k, v, q = inputs(total, 61 + at)
        k[at:at + 16] = key_for(q, -100.0)
        large = v[at:at + 16] * F32(1e20)
        v *= F32(1e-20)
        v[at:at + 16] = large
        attend(fh, k, v, q, total - 1)
