"""A batch's step as it is served: rotations from positions, attention over the prompt that all
sequences share, the layer's projections, the vocabulary head, rules on its logits and the
next tokens, in one captured graph that advances itself, against the same step of the calls
that were there before."""
import numpy as np
import pytest

import gen
from gpu_util import F32, assert_bitwise, host, max_rel, to_dev
from test_gpu_batch_layer import DIM, G, H, int32, layer_of, matrices
from test_gpu_logits import ruled, tokens_of

pytestmark = pytest.mark.gpu
VOCAB = 1003


@pytest.fixture(scope="module")
def fh():
    import focr_hip

    return focr_hip


def frequencies():
    """Time turns the first 16 pairs of every head, a place in the image the others, by directions of each head."""
    rng = np.random.Generator(np.random.PCG64(3))
    f = np.zeros((3, H, 32), F32)
    f[0, :, :16] = 10000.0 ** (-np.arange(16) / 16)
    f[1:, :, 16:] = rng.normal(0, 3, size=(2, H, 16))
    return f


class Served:
    """Sequences behind a common prompt of `shared` positions with an image, one layer, a head."""

    def __init__(self, fh, n, shared=64, page=32, room=64, ctx=None):
        self.fh, self.n, self.shared = fh, n, shared
        m, _ = matrices(fh)
        rng = np.random.Generator(np.random.PCG64(5))
        self.rotary = fh.Rotary(frequencies(), ctx=ctx)
        self.layer = layer_of(fh, m, to_dev(gen.uniform((H,), -2.0, 2.0, 7)), shared, fh.PrefillProjection.I16)
        self.head = fh.Linear.from_f32(rng.normal(0, 0.05, size=(VOCAB, DIM)).astype(F32))
        self.embedding = to_dev(rng.normal(0, 1, size=(VOCAB, DIM)).astype(F32))
        front, back = shared // page, -(-room // page)
        self.pages = fh.KvPages(front + n * back, page, n, front + back, H, G, key_heads=H)
        ids = rng.permutation(front + n * back)
        for i in range(n):
            self.pages.map(i, 0, np.concatenate([ids[:front], ids[front + i * back:front + (i + 1) * back]]))
        # The prompt: an image of 40 positions, then text.
        places = np.zeros((shared, 3), F32)
        places[:, 0] = np.arange(shared)
        places[:40, 1:] = rng.uniform(-1, 1, size=(40, 2))
        h = to_dev(gen.normal((shared, DIM), 1.0, 11))
        self.layer.prefill(h, self.rotary.factors(to_dev(places)), 0, 40)
        self.layer.enter_pages(self.pages, 0)
        self.lens = int32([shared] * n)
        self.positions = to_dev(np.tile(np.array([[shared, 0, 0]], F32), (n, 1)))
        self.history = to_dev(rng.integers(0, VOCAB, size=(n, room)).astype(np.int32))
        self.lengths = int32([3 + i % 5 for i in range(n)])
        bits = rng.random((n, -(-VOCAB // 32) * 32)) < 0.8
        self.rules = fh.LogitRules(history=self.history, lengths=self.lengths, recent=20,
                                   penalties=to_dev(np.array([[1.3, 0.3, 0.1]], F32)),
                                   bias_tokens=to_dev(np.array([[5, 900, 17]], np.int32)), bias=to_dev(np.array([[2.0, -1.0, 0.5]], F32)),
                                   allowed=to_dev(np.packbits(bits, axis=1, bitorder="little").view(np.int32)))
        self.allowed = bits[:, :VOCAB]
        self.max_len = shared + room

    def logits(self, h):
        out = h.new_empty((self.n, VOCAB))
        for at in range(0, self.n, 8):
            self.head.linear(h[at:at + 8].contiguous(), min(8, self.n - at), output=out[at:at + 8])
        return out


@pytest.mark.parametrize("n", [3, 12])
def test_a_step_is_that_of_the_calls_it_replaces(fh, n):
    one, two = Served(fh, n), Served(fh, n)
    h0 = gen.normal((n, DIM), 1.0, 13)
    a, b = to_dev(h0), to_dev(h0)
    one.layer.decode_pages(a, one.rotary.at(one.positions), one.pages, one.lens, one.max_len, shared=one.shared)
    two.layer.decode_pages(b, two.rotary.factors(two.positions), two.pages, two.lens, two.max_len)
    # Attention within FP32 rounding, through the layer: the tolerance of its other tests.
    assert max_rel(host(a), host(b)) <= 1e-4
    assert_bitwise(host(one.layer._buf("pq", (n, H, 64))), host(two.layer._buf("pq", (n, H, 64))), "queries")
    for x, y in zip(*(s.pages.dequantize(n, s.lens) for s in (one, two))):
        assert_bitwise(host(x), host(y), "cache")
    z = one.logits(a)
    want = ruled(host(z), host(one.history), host(one.lengths), 20, host(one.rules.penalties), host(one.rules.bias_tokens),
                 host(one.rules.bias), host(one.rules.allowed))
    assert host(fh.select_tokens(z, n, VOCAB, one.rules)).tolist() == tokens_of(want)
    assert one.pages.refused() == two.pages.refused() == []


def test_a_session_alone_takes_positions_too(fh):
    # Prefill and decode of one session: positions in the place of factors, bitwise.
    m, _ = matrices(fh)
    rotary, got = fh.Rotary(frequencies()), []
    p = gen.normal((40, 3), 20.0, 17)
    for positions in (False, True):
        for kv_bits in (32, 8):
            layer = fh.DecoderLayer(m["qkv"], m["wo"], m["w13"], m["w2"], to_dev(gen.uniform((H,), -2.0, 2.0, 7)), 40, kv_bits=kv_bits)
            of = (lambda x: rotary.at(to_dev(x))) if positions else (lambda x: rotary.factors(to_dev(x)))
            paired = p.copy()
            paired[:, 1:] = 0.0  # the sealed cache shares the temporal halves of paired heads
            h = to_dev(gen.normal((34, DIM), 1.0, 19))
            layer.prefill(h, of(paired[:34]), 0, 10)
            step = to_dev(gen.normal((3, DIM), 1.0, 23))
            layer.decode(step, of(paired[34:37]))
            one = to_dev(gen.normal((1, DIM), 1.0, 29))
            layer.decode(one, of(paired[37:38]))
            got.append([host(x) for x in (h, step, one)])
    for a, b in zip(got[:2], got[2:]):
        for x, y in zip(a, b):
            assert_bitwise(x, y)
    with pytest.raises(fh.FocrError) as e:
        layer.decode(to_dev(np.ones((1, DIM), F32)), fh.Rotary(np.ones((1, 4, 32), F32)).at(to_dev(np.ones((1, 1), F32))))
    assert e.value.code == -2


def test_a_captured_step_advances_itself(fh):
    import torch

    n, steps = 5, 12
    ctx = fh.default_context()
    one, two = Served(fh, n), Served(fh, n)
    tokens = int32([1, 2, 3, 4, 5])
    h = torch.zeros(n, DIM, device="cuda:0")

    def step(s, h, tokens):
        torch.index_select(s.embedding, 0, tokens, out=h)
        s.layer.decode_pages(h, s.rotary.at(s.positions), s.pages, s.lens, s.max_len, shared=s.shared)
        fh.select_tokens(s.logits(h), n, VOCAB, s.rules, tokens=tokens, append=True)
        s.lens.add_(1)
        s.positions[:, 0].add_(1.0)

    # The buffers grow uncaptured; what this step left is taken back.
    kept = [t.clone() for t in (one.history, one.lengths, one.lens, one.positions)]
    step(one, h, int32([1, 2, 3, 4, 5]))
    for t, k in zip((one.history, one.lengths, one.lens, one.positions), kept):
        t.copy_(k)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ctx.use_stream(torch.cuda.current_stream())
        step(one, h, tokens)
    ctx.use_stream(torch.cuda.current_stream())
    eager, state = int32([1, 2, 3, 4, 5]), torch.zeros(n, DIM, device="cuda:0")
    for i in range(steps):
        graph.replay()
        torch.cuda.synchronize()
        got = host(tokens).tolist()
        step(two, state, eager)
        assert_bitwise(host(h), host(state), f"step {i}")
        assert got == host(eager).tolist() and min(got) >= 0
        assert all(one.allowed[r, t] for r, t in enumerate(got))
        for a, b in ((one.history, two.history), (one.lengths, two.lengths), (one.lens, two.lens)):
            assert np.array_equal(host(a), host(b))
    assert host(one.lens).tolist() == [one.shared + steps] * n
    assert one.pages.refused() == two.pages.refused() == []
