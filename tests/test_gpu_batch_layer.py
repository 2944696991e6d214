"""One decoder layer of 4-bit weights serving a batch of sessions from the paged
cache: prefill, entering the pages, steps of one and of several rows a session,
against the same calls made one by one (bitwise) and against a 64-bit layer."""
import numpy as np
import pytest

import gen
from gpu_util import F32, assert_bitwise, host, max_rel, to_dev

pytestmark = pytest.mark.gpu
H, G, DIM, FFN = 16, 8, 192, 256


@pytest.fixture(scope="module")
def fh():
    import focr_hip

    return focr_hip


def matrices(fh, bits=4):
    rng = np.random.Generator(np.random.PCG64(3))
    out, w64 = {}, {}
    for name, n, k in (("qkv", (H + 2 * G) * 64, DIM), ("wo", DIM, H * 64), ("w13", 2 * FFN, DIM), ("w2", DIM, FFN)):
        codes = rng.integers(-8, 8, size=(n, k)).astype(np.int8)
        scales = rng.uniform(0.004, 0.012, size=(n, k // 64)).astype(F32)
        out[name] = fh.QuantLinear.from_parts(n, k, 64, codes, scales, bits=bits)
        w64[name] = codes.astype(np.float64) * np.repeat(scales.astype(np.float64), 64, axis=1)
    return out, w64


def layer_of(fh, m, sinks, capacity, projection):
    return fh.DecoderLayer(m["qkv"], m["wo"], m["w13"], m["w2"], sinks, capacity, projection=projection)


def rope_table(rows, seed, alike=False):
    rng = np.random.Generator(np.random.PCG64(seed))
    angle = rng.uniform(-3.0, 3.0, size=(rows, H, 32))
    if alike:
        angle[:, 1::2] = angle[:, 0::2]
    return np.stack([np.cos(angle), np.sin(angle)], axis=-1).astype(F32)


def int32(values):
    return to_dev(np.asarray(values, dtype=np.int32))


def step64(w, h, attn):
    """The layer after attention, in 64 bits."""
    norm = lambda x: x / np.sqrt((x * x).mean(axis=1, keepdims=True) + 2.0 ** -23)  # noqa: E731
    h = h + attn.reshape(len(h), -1) @ w["wo"].T
    y = norm(h) @ w["w13"].T
    return h + (np.maximum(y[:, 0::2], 0) ** 2 * y[:, 1::2]) @ w["w2"].T


def attention64(q, k, v, first, sinks):
    out = np.empty(q.shape)
    for r in range(len(q)):
        for h in range(H):
            s = k[:first + r + 1, h] @ q[r, h] / 8.0
            p = np.exp(s - s.max())
            out[r, h] = p @ v[:first + r + 1, h // 2] / p.sum() / (1 + np.exp(sinks[h] - s.max() - np.log(p.sum())))
    return out


@pytest.mark.parametrize("sessions,rows,projection", [(3, [1, 1, 1], "I16"), (3, [2, 0, 5], "I16"), (12, [1] * 12, "F32_MFMA"),
                                                      (4, [8, 3, 1, 8], "F32_CHAIN")])
def test_a_batch_of_sessions(fh, sessions, rows, projection):
    import torch

    m, w = matrices(fh)
    sinks_h = gen.uniform((H,), -2.0, 2.0, 5)
    sinks = to_dev(sinks_h)
    kernel = fh.PrefillProjection[projection]
    prompts = [11 + 17 * i % 90 for i in range(sessions)]
    room = max(prompts) + 40
    pages = fh.KvPages(sessions * 9, 16, sessions, -(-room // 16), H, G, key_heads=H)
    free = list(np.random.Generator(np.random.PCG64(7)).permutation(sessions * 9))
    prefix = []
    for i, n in enumerate(prompts):
        pages.map(i, 0, [free.pop() for _ in range(-(-(n + 40) // 16))])
        layer = layer_of(fh, m, sinks, n, kernel)
        h = to_dev(gen.normal((n, DIM), 1.0, 11 + i))
        layer.prefill(h, to_dev(rope_table(n, 31 + i)), 0, n // 2)
        layer.enter_pages(pages, i)
        prefix.append(n)
    layer = layer_of(fh, m, sinks, 8, kernel)
    lens = list(prompts)
    for step in range(3):
        total = sum(rows)
        h0 = gen.normal((total, DIM), 1.0, 101 + step)
        rope = to_dev(rope_table(total, 131 + step))
        row_start = int32(np.concatenate([[0], np.cumsum(rows)]))
        h, alone = to_dev(h0), to_dev(h0)
        stages = []
        layer.decode_pages(h, rope, pages, int32(lens), room, row_start=row_start, clock=stages.append)
        assert stages == ["qkv", "qkv_rows", "attention", "wo", "w13", "w2"]
        q = layer._buf("pq", (total, H, 64)).clone()
        attn = layer._buf("pattn", (total, H, 64)).clone()
        # The same calls one by one; appending the rows again leaves the same cache.
        if total > 8:
            qkv = m["qkv"].prefill(alone, total, row_scale=fh.row_scales(alone, DIM), kernel=kernel)
        else:
            qkv = m["qkv"].linear_ex(alone, total, rms_norm=True)
        assert_bitwise(host(pages.qkv_rows(qkv, rope, int32(lens), row_start=row_start)), host(q), "queries")
        assert_bitwise(host(pages.attention(q, int32(lens), room, row_start=row_start, sinks=sinks)), host(attn), "attention")
        if total > 8:
            m["wo"].prefill(attn, total, epilogue=fh.Epilogue.ADD, out=alone, kernel=kernel)
            gated = m["w13"].prefill(alone, total, row_scale=fh.row_scales(alone, DIM), epilogue=fh.Epilogue.GLU, kernel=kernel)
            m["w2"].prefill(gated, total, epilogue=fh.Epilogue.ADD, out=alone, kernel=kernel)
        else:
            m["wo"].linear_ex(attn, total, epilogue=fh.Epilogue.ADD, out=alone)
            gated = m["w13"].linear_ex(alone, total, rms_norm=True, epilogue=fh.Epilogue.GLU)
            m["w2"].linear_ex(gated, total, epilogue=fh.Epilogue.ADD, out=alone)
        assert_bitwise(host(h), host(alone), "layer")
        # The attention of each session over what the cache holds, and the layer behind it, in 64 bits.
        after = [n + r for n, r in zip(lens, rows)]
        k, v = (host(x).astype(np.float64) for x in pages.dequantize(sum(after), int32([0] * sessions),
                                                                     row_start=int32(np.concatenate([[0], np.cumsum(after)]))))
        at = first = 0
        want = np.empty((total, H, 64))
        for n, r, a in zip(lens, rows, after):
            want[at:at + r] = attention64(host(q)[at:at + r].astype(np.float64), k[first:first + a], v[first:first + a], n, sinks_h)
            at, first = at + r, first + a
        # FP32's tolerance for attention; the layer's as in its other tests. The INT16 panels
        # take their inputs to 2^-15.
        assert max_rel(host(attn), want) <= 1e-5
        loose = 1e-4 if total <= 8 or projection != "I16" else 1e-3
        assert max_rel(host(h), step64(w, h0.astype(np.float64), want)) <= loose
        lens = after
    assert pages.refused() == []
    torch.cuda.synchronize()


def test_refusals(fh):
    m, _ = matrices(fh)
    layer = layer_of(fh, m, to_dev(np.zeros(H, F32)), 20, fh.PrefillProjection.I16)
    pages, narrow = fh.KvPages(4, 16, 2, 1, H, G, key_heads=H), fh.KvPages(4, 16, 2, 2, H, G)
    other = fh.KvPages(4, 16, 2, 2, 8, 4)
    elsewhere = fh.KvPages(4, 16, 2, 2, H, G, ctx=fh.Context(0))
    h, rope = to_dev(np.ones((2, DIM), F32)), to_dev(rope_table(2, 1))

    def refused(code, call):
        with pytest.raises(fh.FocrError) as e:
            call()
        assert e.value.code == code, str(e.value)

    refused(-2, lambda: layer.enter_pages(pages, 0))  # nothing prefilled
    x = to_dev(np.ones((18, DIM), F32))
    layer.prefill(x, to_dev(rope_table(18, 2)), 0, 3)
    refused(-2, lambda: layer.enter_pages(pages, 0))  # one page of 16
    refused(-2, lambda: layer.enter_pages(narrow, 0))
    refused(-2, lambda: layer.enter_pages(other, 0))
    refused(-2, lambda: layer.enter_pages(pages, 2))
    refused(-2, lambda: layer.decode_pages(h, rope, other, int32([0, 0]), 16))
    refused(-1, lambda: layer.decode_pages(h, rope, elsewhere, int32([0, 0]), 16))
    assert layer.decode_pages(h[:0], rope[:0], pages, int32([0, 0]), 16).shape == (0, DIM)


def test_captured_batch_steps(fh):
    # A step of the whole layer in one graph, the lengths advanced by it, as serving replays it.
    import torch

    m, _ = matrices(fh)
    ctx = fh.default_context()
    sinks = to_dev(gen.uniform((H,), -2.0, 2.0, 5))
    n, steps = 5, 20
    caches = []
    for _ in range(2):
        pages = fh.KvPages(n * 2, 32, n, 2, H, G)
        for i in range(n):
            pages.map(i, 0, [2 * i + 1, 2 * i])
        caches.append(pages)
    layer = layer_of(fh, m, sinks, 8, fh.PrefillProjection.I16)
    h, lens = torch.zeros(n, DIM, device="cuda:0"), int32([3, 0, 30, 15, 9])
    rope = to_dev(rope_table(n, 3, alike=True))
    start = host(lens).copy()
    for pages in caches:
        k, v = gen.normal((30 * n, G, 64), 1.0, 9), gen.normal((30 * n, G, 64), 1.0, 10)
        pages.append(to_dev(k), to_dev(v), int32([0] * n), row_start=int32([30 * i for i in range(n + 1)]))
    layer.decode_pages(torch.zeros(n, DIM, device="cuda:0"), rope, caches[1], int32(start), 64)  # the buffers grow uncaptured
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ctx.use_stream(torch.cuda.current_stream())
        layer.decode_pages(h, rope, caches[0], lens, 64)
        lens.add_(1)
    ctx.use_stream(torch.cuda.current_stream())
    for step in range(steps):
        x = gen.normal((n, DIM), 1.0, 200 + step)
        h.copy_(to_dev(x))
        graph.replay()
        torch.cuda.synchronize()
        got = host(h)
        want = layer.decode_pages(to_dev(x), rope, caches[1], int32(start + step), 64)
        assert_bitwise(got, host(want), f"step {step}")


def test_a_captured_step_keeps_its_buffers(fh):
    # A larger batch in between must not leave the graph writing memory that others have.
    import torch

    m, _ = matrices(fh)
    ctx = fh.default_context()
    layer = layer_of(fh, m, to_dev(np.zeros(H, F32)), 8, fh.PrefillProjection.I16)
    n = 7
    caches = [fh.KvPages(n, 16, n, 1, H, G) for _ in range(2)]
    for pages in caches:
        for i in range(n):
            pages.map(i, 0, [i])
    rope = to_dev(rope_table(n, 3, alike=True))
    x = gen.normal((n, DIM), 1.0, 11)
    zeros = int32([0] * n)
    layer.decode_pages(to_dev(x[:2]), rope[:2], caches[1], zeros[:2], 16)
    h = torch.zeros(2, DIM, device="cuda:0")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ctx.use_stream(torch.cuda.current_stream())
        layer.decode_pages(h, rope[:2], caches[0], zeros[:2], 16)
    ctx.use_stream(torch.cuda.current_stream())
    layer.decode_pages(to_dev(x), rope, caches[1], zeros, 16)
    others = [torch.full((2, w), 7.0, device="cuda:0") for w in ((H + 2 * G) * 64, H * 64, H * 64, FFN) for _ in range(4)]
    want = host(layer.decode_pages(to_dev(x[:2]), rope[:2], caches[1], zeros[:2], 16))
    for step in range(3):
        h.copy_(to_dev(x[:2]))
        graph.replay()
        torch.cuda.synchronize()
        assert_bitwise(host(h), want, f"replay {step}")
    assert all((host(t) == 7.0).all() for t in others)


def test_entering_on_another_stream(fh):
    # The context runs on its own stream, the batch's arrays are made on torch's.
    import torch

    m, _ = matrices(fh)
    got = []
    for own in (False, True):
        ctx = fh.Context(0)
        layer = fh.DecoderLayer(m["qkv"], m["wo"], m["w13"], m["w2"], to_dev(np.zeros(H, F32)), 40, ctx=ctx)
        pages = fh.KvPages(6, 16, 2, 3, H, G, key_heads=H, ctx=ctx)
        pages.map(1, 0, [4, 2, 5])
        layer.prefix_k[:40] = to_dev(gen.normal((40, H, 64), 1.0, 21))
        layer.v[:40] = to_dev(gen.normal((40, G, 64), 1.0, 22))
        layer.len = layer.prefix_len = 40
        torch.cuda.synchronize()
        if own:
            ctx.use_stream(None)
        layer.enter_pages(pages, 1)
        junk = [torch.full((n,), 1 << 28, dtype=torch.int32, device="cuda:0") for n in (2, 3, 2, 3)]
        ctx.sync()
        assert len(junk) == 4 and pages.refused() == []
        ctx.use_stream(torch.cuda.current_stream())
        got.append([host(t) for t in pages.dequantize(40, int32([-1, 0]), row_start=int32([0, 0, 40]))])
        with pytest.raises(fh.FocrError) as e:
            layer.enter_pages(fh.KvPages(6, 16, 2, 3, H, G, key_heads=H), 1)  # of another context
        assert e.value.code == -1
    for a, b in zip(*got):
        assert_bitwise(a, b)
