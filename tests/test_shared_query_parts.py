"""How far the two FP16 parts that attention over a shared prefix takes of a query's elements are
from them, restated in NumPy, against what the header says."""
import re
from pathlib import Path

import numpy as np
import pytest

F32 = np.float32


def stated():
    """Exponents of the bound: of an element, of the largest one, and where that is tiny."""
    text = " ".join((Path(__file__).resolve().parents[1] / "include" / "focr_hip.h").read_text().replace("\n *", "\n").split())
    m = re.search(r"elements are taken to 2\^-(\d+) of themselves, and 2\^-(\d+) of its largest(?: \(2\^-(\d+) where that is below 2\^-(\d+)\))?", text)
    return [int(x) if x else None for x in m.groups()]


def parts(q):
    """A query [n] as the sum of its parts, in 64 bits."""
    _, e = np.frexp(np.abs(q).max())
    e = max(int(e), -90)
    scaled = np.ldexp(q, 14 - e).astype(F32)
    high = scaled.astype(np.float16)
    low = (scaled - high.astype(F32)).astype(np.float16)
    return np.ldexp(high.astype(np.float64) + low.astype(np.float64), e - 14)


def queries():
    rng = np.random.Generator(np.random.PCG64(3))
    yield np.array([1.0002443, 1.0, 1.9999999], F32)  # an odd rest between 2^11 and 2^12 units
    yield np.array([1.0, 2.0 ** -24 * 1.4999999, -(2.0 ** -30) * 1.9, 2.0 ** -38 * 0.999, 2.0 ** -37 * 1.01], F32)
    for spread in (0, 4, 12, 24, 40, 100):
        for top in (0, 60, 126, -60, -90, -91, -100, -125):
            q = rng.uniform(1, 2, 20000) * rng.choice([-1, 1], 20000) * 2.0 ** (top - rng.uniform(0, spread, 20000))
            yield q.astype(F32)
    for _ in range(2000):
        yield rng.normal(0, 1, 64).astype(F32)


def test_the_header_states_what_the_parts_lose():
    own, top, tiny, below = stated()
    worst = [0.0, 0.0]
    for q in queries():
        off, x, most = np.abs(parts(q) - q.astype(np.float64)), np.abs(q.astype(np.float64)), np.abs(q.astype(np.float64)).max()
        least = 2.0 ** -tiny if tiny and most < 2.0 ** -below else 2.0 ** -top * most
        over = off > np.maximum(2.0 ** -own * x, least)
        assert not over.any(), f"{q[over][:4]} beside {most}: {off[over][:4]}"
        if most >= 2.0 ** -91:
            near = x > 2.0 ** -13 * most
            worst[0] = max(worst[0], float((off[near] / x[near]).max()))
            worst[1] = max(worst[1], float(off[~near].max(initial=0) / most))
    # And no less than that is lost.
    assert worst[0] > 2.0 ** -own * 0.99 and worst[1] > 2.0 ** -top * 0.9
