"""One element of a query at a time through attention over a shared prefix: how far its score may be
off, with the other roundings too small to cover it."""
import math

import numpy as np
import pytest

import gen
from gpu_util import F32, host, to_dev
from test_gpu_pages import int32

pytestmark = pytest.mark.gpu
HEADS, KEYS = 16, 64


@pytest.fixture(scope="module")
def fh():
    import focr_hip

    return focr_hip


def elements(n, seed):
    """[n] in 1 .. 2: any, and those whose rest after 11 bits is odd and above 2^11 units, which lose a unit."""
    rng = np.random.Generator(np.random.PCG64(seed))
    x = rng.uniform(1, 2, n).astype(F32)
    units = rng.integers(1 << 10, 1 << 11, n // 2) * 8192 + rng.integers(2050, 4094, n // 2) // 2 * 2 + 1
    x[:n // 2] = np.ldexp(units.astype(np.float64), -23).astype(F32)
    return np.minimum(x, F32(2 - 2.0 ** -23))


@pytest.mark.parametrize("beside", [0, 10, 16, 20])
@pytest.mark.parametrize("sequences", [2, 70])
def test_one_element_of_a_query(fh, sequences, beside):
    # Key 3's score is 32 times the element x, key 0's, like all others', 0; the value is key 0's alone:
    #   out = v0 / (e^(32 x) + 64).
    # Codes are 127 and 64 at scales that are powers of two, so products and sums are exact; the
    # largest score is rounded once, the others' exponent is that number and its own exponent what the
    # rounding took, so it cancels. Off are: the element, and the constant log2(e) / 8 in FP32 (both times
    # 32 x, as a share of the result), two exponentials by a unit of 2^-23 each, and six roundings of
    # 2^-24 (value's parts, the sums, the division). With `beside`, an element 2^beside times
    # as large meets no key, and x may be off by 2^-38 of that too (the large one is below 2^(beside + 1)).
    page, n = 64, sequences
    kv = fh.KvPages(1 + n, page, n + 1, 2, HEADS, HEADS, key_heads=HEADS)
    kv.map(n, 0, [n])
    for i in range(n):
        kv.map(i, 1, [i])
    k, v = np.zeros((KEYS + n, HEADS, 64), F32), np.zeros((KEYS + n, HEADS, 64), F32)
    k[n + 3, :, 0], k[n + 5, :, 2] = 256.0, 508.0
    v[n] = 127.0 / 128.0
    kv.append(to_dev(k), to_dev(v), int32([KEYS] * n + [0]), row_start=int32(list(range(n + 1)) + [n + KEYS]))
    gk, gv = (host(t) for t in kv.dequantize(KEYS, int32([-1] * n + [0]), row_start=int32([0] * (n + 1) + [KEYS])))
    assert (gk[3, :, 0] == 256.0).all() and (gk[5, :, 2] == 508.0).all() and np.count_nonzero(gk) == 2 * HEADS
    assert (gv[0] == 127.0 / 128.0).all() and np.count_nonzero(gv) == HEADS * 64
    x = elements(n * HEADS, 7 + beside).reshape(n, HEADS)
    q = np.zeros((n, HEADS, 64), F32)
    q[:, :, 0] = x
    if beside:
        q[:, :, 1] = gen.uniform((n, HEADS), 1.0, 2.0, 11) * F32(2.0 ** beside)
    got = host(kv.attention_shared(to_dev(q), int32([KEYS] * n), KEYS + 1, KEYS, n)).astype(np.float64)
    assert kv.refused() == []
    score = 32.0 * x.astype(np.float64)
    want = 127.0 / 128.0 / (np.exp(score) + 64.0)
    constant = abs(float(F32(0.180336880111120426)) * 8.0 * math.log(2.0) - 1.0)
    share = constant + 2.0 ** -23 + (2.0 ** (beside + 1 - 38) if beside else 0.0)
    bound = np.expm1(score * share) + 2 * 2.0 ** -23 + 6 * 2.0 ** -24
    off = np.abs(got / want[:, :, None] - 1.0).max(axis=2)
    assert (off <= bound).all(), f"{(off / bound).max()} times what is allowed, at an element of {x[np.unravel_index((off / bound).argmax(), x.shape)]}"
    if not beside:
        # A lost unit is 2^-23 of an element near 1 and 2^-24 of one near 2: near 1 the test tells the two bounds apart.
        less = np.expm1(score * (constant + 2.0 ** -24)) + 2 * 2.0 ** -23 + 6 * 2.0 ** -24
        assert (off > less).any()
