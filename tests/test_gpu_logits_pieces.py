"""Rules on logits where a workgroup has a row's pieces one after another, and lists of biases longer
than what it holds."""
import numpy as np
import pytest

from gpu_util import F32
from test_gpu_logits import mask_of, rules_of, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fh():
    import focr_hip

    return focr_hip


@pytest.mark.parametrize("rows,vocab,at", [(1025, 8193, 0), (1030, 16390, 1), (1100, 16387, 3), (1025, 24577, 2)])
def test_several_pieces_of_a_workgroup(fh, rows, vocab, at):
    # More rows than the context has words for: a row is one workgroup's, in pieces of 8,192 tokens.
    rng = np.random.Generator(np.random.PCG64(rows + vocab))
    logits = rng.normal(0, 3, size=(rows, vocab)).astype(F32)
    rules = rules_of(rng, rows, vocab, 60, 20)
    run(fh, logits, rules | dict(recent=40), at=at)


@pytest.mark.parametrize("where", [0, 8191, 8192, 16383, 16389])
def test_ties_over_pieces(fh, where):
    # The same largest value at the ends of pieces; the lowest allowed one is taken.
    rows, vocab = 1027, 16390
    rng = np.random.Generator(np.random.PCG64(where))
    logits = rng.integers(-3, 3, size=(rows, vocab)).astype(F32)
    logits[:, [where, 16389]] = 7.0
    run(fh, logits, {})
    bits = rng.random((rows, vocab)) < 0.5
    bits[::2, where] = False
    bits[3::4, :8192] = False
    bits[5] = False
    run(fh, logits, dict(allowed=mask_of(bits)), at=1)


def test_a_piece_that_is_not_finite(fh):
    rows, vocab = 1025, 20000
    rng = np.random.Generator(np.random.PCG64(5))
    logits = rng.normal(0, 3, size=(rows, vocab)).astype(F32)
    logits[np.arange(0, 1000, 10), rng.integers(0, vocab, 100)] = np.nan
    logits[np.arange(1, 1000, 10), rng.integers(0, vocab, 100)] = np.inf
    logits[2, :] = -np.inf
    logits[3, :16384] = -np.inf
    run(fh, logits, {}, at=2)


@pytest.mark.parametrize("n_bias", [1023, 1024, 1025, 5000, 16383])
@pytest.mark.parametrize("rows,vocab,alike", [(3, 5000, False), (9, 20011, True), (2, 9000, False)])
def test_more_biases_than_are_held(fh, n_bias, rows, vocab, alike):
    # Tokens that come twice, on either side of the 1,024th entry, and entries that are none.
    rng = np.random.Generator(np.random.PCG64(n_bias + rows))
    logits = rng.normal(0, 3, size=(rows, vocab)).astype(F32)
    rules = rules_of(rng, rows, vocab, 50, n_bias, alike=alike)
    tokens = rules["bias_tokens"]
    tokens[:, -1] = tokens[:, 0] = 4  # the last counts
    tokens[:, 1] = tokens[:, n_bias // 2] = vocab - 1
    tokens[:, -3:-1] = [-1, vocab]
    run(fh, logits, rules)
    run(fh, logits, {k: rules[k] for k in ("bias_tokens", "bias")}, at=3)


def test_long_lists_over_pieces(fh):
    rows, vocab = 1026, 8200
    rng = np.random.Generator(np.random.PCG64(7))
    logits = rng.normal(0, 3, size=(rows, vocab)).astype(F32)
    run(fh, logits, rules_of(rng, rows, vocab, 30, 2000, alike=True))
