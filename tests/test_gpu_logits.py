"""Penalties, biases and masks on logits with the greedy token, against the rules restated in
NumPy with FP32 steps: bitwise."""
import numpy as np
import pytest

import gen
from gpu_util import F32, assert_bitwise, host, to_dev

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fh():
    import focr_hip

    return focr_hip


def ruled(logits, history=None, lengths=None, recent=0, penalties=None, bias_tokens=None, bias=None, allowed=None):
    """The logits under the rules, every step in FP32."""
    z = logits.copy()
    rows, vocab = z.shape
    of = lambda t, r: t[0 if len(t) == 1 else r]  # noqa: E731
    with np.errstate(all="ignore"):
        for r in range(rows):
            if penalties is not None:
                n = min(max(int(lengths[r]), 0), history.shape[1])
                seen = history[r, max(0, n - recent) if recent else 0:n]
                seen = seen[(seen >= 0) & (seen < vocab)]
                tokens, counts = np.unique(seen, return_counts=True)
                repetition, presence, frequency = (F32(x) for x in of(penalties, r))
                x = z[r, tokens]
                x = np.where(x > 0, (x / repetition).astype(F32), (x * repetition).astype(F32))
                z[r, tokens] = x - ((counts.astype(F32) * frequency).astype(F32) + presence).astype(F32)
            if bias is not None:
                last = {int(t): b for t, b in zip(of(bias_tokens, r), of(bias, r)) if 0 <= t < vocab}
                for t, b in last.items():
                    z[r, t] = F32(z[r, t] + b)
            if allowed is not None:
                bits = np.unpackbits(of(allowed, r).view(np.uint8), bitorder="little")[:vocab]
                z[r, bits == 0] = -np.inf
    return z


def tokens_of(z):
    out = []
    for row in z:
        if np.isnan(row).any() or (row == np.inf).any():
            out.append(-2)
        else:
            out.append(-1 if (row == -np.inf).all() else int(np.argmax(row)))  # the first of equal ones
    return out


def mask_of(bits):
    """bool [rows][vocab] to int32 [rows][ceil(vocab / 32)]; bits behind the vocabulary are set, and do not count."""
    rows, vocab = bits.shape
    full = np.ones((rows, -(-vocab // 32) * 32), bool)
    full[:, :vocab] = bits
    return np.packbits(full, axis=1, bitorder="little").view(np.int32)


def rules_of(rng, rows, vocab, cap, n_bias, alike=False):
    """Every rule at once: histories of any length with tokens that come often and entries that are none."""
    own = 1 if alike else rows
    history = rng.integers(0, min(vocab, 50), size=(rows, cap)).astype(np.int32)
    wide = rng.random(history.shape) < 0.5
    history[wide] = rng.integers(-3, vocab + 3, size=int(wide.sum()))
    lengths = rng.integers(0, cap + 1, size=rows).astype(np.int32)
    lengths[0] = cap + 5
    if rows > 2:
        lengths[1:3] = [0, -4]
    penalties = np.stack([rng.uniform(0.7, 2.0, own), rng.uniform(-1, 2, own), rng.uniform(-0.1, 0.5, own)], axis=1).astype(F32)
    tokens = rng.integers(-2, vocab + 2, size=(own, n_bias)).astype(np.int32)
    return dict(history=history, lengths=lengths, penalties=penalties, bias_tokens=tokens,
                bias=rng.normal(0, 4, size=(own, n_bias)).astype(F32), allowed=mask_of(rng.random((own, vocab)) < 0.7))


def given(fh, rules):
    return fh.LogitRules(**{k: to_dev(v) if isinstance(v, np.ndarray) else v for k, v in rules.items()})


def run(fh, logits, rules, label="", at=0):
    """Tokens alone, tokens with the logits, and the logits alone; `at`: floats before the logits."""
    import torch

    rows, vocab = logits.shape
    place = torch.full((rows * vocab + at + 9,), 7.0, device="cuda:0")
    x = place[at:at + rows * vocab].view(rows, vocab)
    x.copy_(to_dev(logits))
    want = ruled(logits, **rules)
    r = given(fh, rules)
    assert host(fh.select_tokens(x, rows, vocab, r)).tolist() == tokens_of(want), label
    for shift in (at, at + 1):  # the results on the same place of a line of memory, and on another
        out = torch.full((rows * vocab + shift + 9,), 9.0, device="cuda:0")
        y = out[shift:shift + rows * vocab].view(rows, vocab)
        assert host(fh.select_tokens(x, rows, vocab, r, adjusted=y)).tolist() == tokens_of(want), label
        assert_bitwise(host(y), want, label)
        assert (host(out)[:shift] == 9.0).all() and (host(out)[shift + rows * vocab:] == 9.0).all()
    assert_bitwise(host(fh.adjust_logits(x, rows, vocab, r)), want, label)
    assert_bitwise(host(x), logits, label)
    assert host(fh.select_tokens(x, rows, vocab, r, adjusted=x)).tolist() == tokens_of(want), label
    assert_bitwise(host(x), want, label)
    assert (host(place)[:at] == 7.0).all() and (host(place)[at + rows * vocab:] == 7.0).all()


@pytest.mark.parametrize("rows", [1, 2, 3, 7])
@pytest.mark.parametrize("vocab", [1, 2, 3, 4, 5, 31, 32, 33, 255, 1003, 1024, 4096, 8191, 8193, 40005])
def test_every_rule(fh, rows, vocab):
    rng = np.random.Generator(np.random.PCG64(rows * 100003 + vocab))
    for at, recent in ((0, 0), (1, 17), (2, 0), (3, 1)):
        logits = rng.normal(0, 3, size=(rows, vocab)).astype(F32)
        rules = rules_of(rng, rows, vocab, 90, 12, alike=at == 3)
        run(fh, logits, rules | dict(recent=recent), f"{at} floats before", at)


@pytest.mark.parametrize("rows,vocab", [(64, 65536), (513, 20003), (512, 4097), (1, 262144), (1, 1000003), (30, 65537)])
def test_large_calls(fh, rows, vocab):
    rng = np.random.Generator(np.random.PCG64(rows + vocab))
    logits = rng.normal(0, 3, size=(rows, vocab)).astype(F32)
    rules = rules_of(rng, rows, vocab, 700, 300)
    run(fh, logits, rules, at=rows % 4)


@pytest.mark.parametrize("only", ["penalties", "bias", "allowed", None])
@pytest.mark.parametrize("rows,vocab", [(3, 5000), (2, 70001)])
def test_each_rule_alone(fh, only, rows, vocab):
    rng = np.random.Generator(np.random.PCG64(11))
    logits = rng.normal(0, 3, size=(rows, vocab)).astype(F32)
    rules = rules_of(rng, rows, vocab, 400, 50)
    keep = {"penalties": ["history", "lengths", "penalties"], "bias": ["bias_tokens", "bias"], "allowed": ["allowed"], None: []}[only]
    run(fh, logits, {k: rules[k] for k in keep})


def test_long_histories_of_one_token(fh):
    # Every entry the same, and all different ones: the counts are whole.
    rng = np.random.Generator(np.random.PCG64(13))
    rows, vocab, cap = 2, 30000, 100000
    history = np.full((rows, cap), 777, np.int32)
    history[1] = rng.permutation(cap) % vocab
    rules = dict(history=history, lengths=np.full(rows, cap, np.int32), penalties=np.array([[1.0, 0.5, 1e-3]], F32))
    logits = rng.normal(0, 3, size=(rows, vocab)).astype(F32)
    run(fh, logits, rules)
    run(fh, logits, rules | dict(recent=99999))


def test_ties_take_the_lowest_index(fh):
    rng = np.random.Generator(np.random.PCG64(17))
    for vocab in (7, 5000, 66000):
        logits = rng.integers(-3, 4, size=(9, vocab)).astype(F32)  # most values come often
        logits[1] = 0.0
        logits[2] = -0.0
        logits[2, vocab // 2] = 0.0
        run(fh, logits, {})
        run(fh, logits, dict(allowed=mask_of(rng.random((9, vocab)) < 0.3)))


def test_rows_without_a_token_and_what_is_not_finite(fh):
    rng = np.random.Generator(np.random.PCG64(19))
    for vocab in (33, 9001):
        logits = rng.normal(0, 3, size=(10, vocab)).astype(F32)
        bits = rng.random((10, vocab)) < 0.5
        bits[:, 5], bits[:, 6] = True, False
        bits[0] = False  # nothing is allowed
        logits[0, 3] = np.nan
        logits[1, 6], logits[2, 6], logits[3, 6] = np.nan, np.inf, -np.inf  # in masked places: no matter
        logits[4, 5], logits[5, 5], logits[6, 5] = np.nan, np.inf, -np.inf  # in allowed ones
        logits[7] = -np.inf
        logits[8] = np.finfo(F32).min
        bits[9] = False
        bits[9, vocab - 1] = True
        logits[9, vocab - 1] = np.finfo(F32).min
        want = tokens_of(ruled(logits, allowed=mask_of(bits)))
        assert want[0] == want[7] == -1 and want[4] == want[5] == -2 and want[9] == vocab - 1 and min(want[1:4]) >= 0
        run(fh, logits, dict(allowed=mask_of(bits)))
    # Rules that leave the range of FP32: infinities are found where they arise.
    logits = np.full((4, 100), -3.0, F32)
    logits[:, 7] = 1.0
    history, lengths = np.full((4, 1), 7, np.int32), np.ones(4, np.int32)
    penalties = np.array([[0.0, 0.0, 0.0], [1.0, -3e38, -3e38], [1.0, 3e38, 3e38], [np.nan, 0.0, 0.0]], F32)
    want = tokens_of(ruled(logits, history, lengths, penalties=penalties))
    assert want == [-2, -2, 0, -2]
    run(fh, logits, dict(history=history, lengths=lengths, penalties=penalties))


def test_a_token_with_every_rule_and_a_bias_twice(fh):
    logits = np.array([[1.0, 2.0, -2.0, 0.5]], F32)
    rules = dict(history=np.array([[1, 2, 1, 9, -1]], np.int32), lengths=np.array([5], np.int32),
                 penalties=np.array([[2.0, 0.25, 0.125]], F32), bias_tokens=np.array([[2, 1, 2, 3]], np.int32),
                 bias=np.array([[100.0, 1.5, 4.0, 0.0]], F32))
    want = np.array([[1.0, 2.0 / 2 - 0.5 + 1.5, -4.0 - 0.375 + 4.0, 0.5]], F32)
    assert_bitwise(ruled(logits, **rules), want)
    run(fh, logits, rules)


def test_captured_steps_append_their_tokens(fh):
    # A greedy loop in one graph: the token goes behind the history, which the next replay counts.
    import torch

    rng = np.random.Generator(np.random.PCG64(23))
    for rows, vocab in ((3, 70000), (1, 500), (600, 333)):
        ctx = fh.Context(0)
        cap, steps = 40, 12
        history = rng.integers(0, vocab, size=(rows, cap)).astype(np.int32)
        lengths = rng.integers(0, 20, size=rows).astype(np.int32)
        lengths[0] = cap - 3  # it fills up
        rules = dict(history=history, lengths=lengths, recent=25, penalties=np.array([[1.3, 0.4, 0.2]], F32))
        r = given(fh, rules)
        logits, tokens = torch.zeros(rows, vocab, device="cuda:0"), torch.zeros(rows, dtype=torch.int32, device="cuda:0")
        fh.select_tokens(logits, rows, vocab, given(fh, rules), ctx=ctx)  # the scratch grows uncaptured
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            ctx.use_stream(torch.cuda.current_stream())
            fh.select_tokens(logits, rows, vocab, r, tokens=tokens, append=True, ctx=ctx)
        ctx.use_stream(torch.cuda.current_stream())
        base = rng.normal(0, 1, size=(rows, vocab)).astype(F32)
        for step in range(steps):
            x = base + rng.normal(0, 0.05, size=(rows, vocab)).astype(F32)
            if step == 4:
                x[0, 2] = np.nan  # no token: nothing is appended
            logits.copy_(to_dev(x))
            graph.replay()
            torch.cuda.synchronize()
            want = tokens_of(ruled(x, **rules))
            assert host(tokens).tolist() == want, f"step {step}"
            for i, t in enumerate(want):
                if t >= 0 and lengths[i] < cap:
                    history[i, lengths[i]] = t
                    lengths[i] += 1
            assert np.array_equal(host(r.lengths), lengths) and np.array_equal(host(r.history), history)
        assert lengths[0] == cap


def test_appending_without_penalties(fh):
    logits = gen.normal((5, 2000), 1.0, 29)
    r = fh.LogitRules(history=to_dev(np.full((5, 3), -1, np.int32)), lengths=to_dev(np.array([0, 1, 2, 3, -1], np.int32)))
    want = tokens_of(logits)
    assert host(fh.select_tokens(to_dev(logits), 5, 2000, r, append=True)).tolist() == want
    assert host(r.lengths).tolist() == [1, 2, 3, 3, -1]
    held = np.full((5, 3), -1, np.int32)
    held[0, 0], held[1, 1], held[2, 2] = want[:3]
    assert np.array_equal(host(r.history), held)


def test_equals_argmax(fh):
    logits = gen.normal((6, 65536), 3.0, 31)
    x = to_dev(logits)
    assert host(fh.select_tokens(x, 6, 65536)).tolist() == fh.argmax(x, 6, 65536)


def test_two_contexts_at_once(fh):
    import torch

    rng = np.random.Generator(np.random.PCG64(37))
    sets = []
    for i in range(2):
        logits = rng.normal(0, 3, size=(40, 50001)).astype(F32)
        rules = rules_of(rng, 40, 50001, 300, 20)
        sets.append((fh.Context(0), torch.cuda.Stream(), to_dev(logits), given(fh, rules), tokens_of(ruled(logits, **rules))))
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (ctx, stream, x, r, _w) in enumerate(sets):
            with torch.cuda.stream(stream):
                ctx.use_stream(stream)
                got[i].append(fh.select_tokens(x, 40, 50001, r, ctx=ctx))
    torch.cuda.synchronize()
    for g, s in zip(got, sets):
        assert all(host(t).tolist() == s[4] for t in g)


def test_refusals(fh):
    import torch

    def refused(code, call):
        with pytest.raises(fh.FocrError) as e:
            call()
        assert e.value.code == code, str(e.value)

    x = to_dev(gen.normal((4, 100), 1.0, 41))
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda:0")  # noqa: E731
    f32 = lambda *shape: torch.zeros(shape, device="cuda:0")  # noqa: E731
    R, select = fh.LogitRules, lambda rules=fh.LogitRules(), **kw: fh.select_tokens(x, 4, 100, rules, **kw)  # noqa: E731
    refused(-2, lambda: fh.select_tokens(x, 4, 99))
    refused(-2, lambda: fh.select_tokens(x[:, ::2], 4, 50))
    refused(-2, lambda: fh.select_tokens(x.half(), 4, 100))
    refused(-1, lambda: fh.select_tokens(x.cpu(), 4, 100, tokens=i32(4)))
    refused(-2, lambda: fh.select_tokens(f32(0, 0), 4, 0))
    refused(-2, lambda: select(tokens=i32(3)))
    refused(-2, lambda: select(tokens=f32(4)))
    refused(-2, lambda: select(adjusted=f32(4, 99)))
    refused(-1, lambda: fh.select_tokens(x[:2], 2, 100, adjusted=x.view(-1)[100:300]))  # partly the same memory
    refused(-1, lambda: select(append=True))
    refused(-1, lambda: select(R(penalties=f32(4, 3))))
    refused(-2, lambda: select(R(history=i32(4, 9))))
    refused(-2, lambda: select(R(history=i32(3, 9), lengths=i32(4))))
    refused(-2, lambda: select(R(history=i32(4, 9), lengths=i32(3))))
    refused(-2, lambda: select(R(history=i32(4, 9).long(), lengths=i32(4))))
    refused(-1, lambda: select(R(lengths=i32(4))))
    history = dict(history=i32(4, 9), lengths=i32(4))
    refused(-2, lambda: select(R(**history, recent=-1)))
    refused(-2, lambda: select(R(**history, penalties=f32(2, 3))))
    refused(-2, lambda: select(R(**history, penalties=f32(4, 2))))
    refused(-2, lambda: select(R(history=i32(4, 1 << 18), lengths=i32(4), penalties=f32(1, 3))))
    refused(-1, lambda: select(R(bias=f32(4, 2))))
    refused(-2, lambda: select(R(bias=f32(4, 2), bias_tokens=i32(4, 3))))
    refused(-2, lambda: select(R(bias=f32(3, 2), bias_tokens=i32(3, 2))))
    refused(-2, lambda: select(R(bias=f32(1, 1 << 14), bias_tokens=i32(1, 1 << 14))))
    refused(-2, lambda: select(R(allowed=i32(4, 3))))
    refused(-2, lambda: select(R(allowed=i32(2, 4))))
    assert select(R(history=i32(4, 1 << 18), lengths=i32(4), penalties=f32(1, 3), recent=9)).shape == (4,)
    assert select(R(bias=f32(4, 0), bias_tokens=i32(4, 0))).shape == (4,)
    assert fh.select_tokens(x[:0], 0, 100).shape == (0,)
