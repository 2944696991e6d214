"""Steps of more than eight rows: a layer whose prompts take the INT16 panels decodes in
FP32 there too, so that a session's step is the same to FP32's rounding whoever else
takes part."""
import numpy as np
import pytest

import gen
from gpu_util import assert_bitwise, host, max_rel, to_dev
from test_gpu_batch_layer import DIM, G, H, int32, layer_of, matrices, rope_table

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fh():
    import focr_hip

    return focr_hip


def steps(fh, kernel, batches, bits=4, **kw):
    """One step of 40 sessions, dealt out in batches of so many: the rows of h after it, and
    the keys and values that the cache then holds of each session, [40][21 x 8 x 64] each."""
    m, _ = matrices(fh, bits)
    n = 40
    layer = layer_of(fh, m, to_dev(gen.uniform((H,), -2.0, 2.0, 5)), 8, kernel)
    pages = fh.KvPages(n * 2, 16, n, 2, H, G)
    for i in range(n):
        pages.map(i, 0, [2 * i + 1, 2 * i])
    k, v = gen.normal((20 * n, G, 64), 1.0, 9), gen.normal((20 * n, G, 64), 1.0, 10)
    pages.append(to_dev(k), to_dev(v), int32([0] * n), row_start=int32([20 * i for i in range(n + 1)]))
    rope = rope_table(n, 3, alike=True)
    x, out, at = gen.normal((n, DIM), 1.0, 11), [], 0
    for size in batches:
        lens, starts = [-1] * n, [min(max(i - at, 0), size) for i in range(n + 1)]
        lens[at:at + size] = [20] * size
        h = to_dev(x[at:at + size])
        layer.decode_pages(h, to_dev(rope[at:at + size]), pages, int32(lens), 32, row_start=int32(starts), **kw)
        out.append(host(h))
        at += size
    assert pages.refused() == []
    held = pages.dequantize(21 * n, int32([0] * n), row_start=int32([21 * i for i in range(n + 1)]))
    return (np.concatenate(out), *(host(x).reshape(n, -1) for x in held))


@pytest.mark.parametrize("bits", [4, 8])
def test_a_sessions_step_does_not_depend_on_the_others(fh, bits):
    # FP32 sums in another order: outputs within 1e-5 of the largest one, the tolerance of FP32's
    # attention, where INT16 activations alone are off by some 1e-4. That is so for a session
    # whose cache is the same to FP32's rounding. A key or value next to the border of two codes may
    # take the other one: it is then off by a step of its block, 1/127 of the block's largest (at most
    # 5 here: normal values, unit heads turned), and so is what attends to it, 1/127 / 21 of 3 and more.
    # A value of some 1 that is off by FP32's 1e-6 at most lies that near a border of steps of 0.02 with a
    # chance of 1e-4, one of a session's 1,024 new ones with 0.1: 16 of 40 sessions are far beyond.
    few, few_k, few_v = steps(fh, fh.PrefillProjection.I16, [8] * 5, bits)
    for batches in ([9, 31], [40], [32, 7, 1]):
        many, k, v = steps(fh, fh.PrefillProjection.I16, batches, bits)
        off = np.maximum(np.abs(k - few_k).max(axis=1), np.abs(v - few_v).max(axis=1))
        assert off.max() <= 5 / 127 * 1.01
        same = off <= 1e-5
        assert same.sum() >= 24
        assert max_rel(many[same], few[same]) <= 1e-5


def test_the_projection_is_the_callers(fh):
    p = fh.PrefillProjection
    h = lambda kernel, **kw: steps(fh, kernel, [40], **kw)[0]  # noqa: E731
    assert_bitwise(h(p.I16), h(p.F32_MFMA))
    assert_bitwise(h(p.F32_CHAIN), h(p.I16, projection=p.F32_CHAIN))
    assert not np.array_equal(h(p.F32_MFMA, projection=p.I16), h(p.F32_MFMA))
