"""A captured decode from positions, replayed after a longer prompt has been through the layer."""
import numpy as np
import pytest

import gen
from gpu_util import assert_bitwise, host, to_dev
from test_gpu_batch_layer import DIM, H, layer_of, matrices
from test_gpu_served_step import frequencies

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fh():
    import focr_hip

    return focr_hip


@pytest.mark.parametrize("rows", [1, 3])
def test_a_longer_prompt_between_a_captured_decode_and_its_replay(fh, rows):
    import torch

    m, _ = matrices(fh)
    ctx, rotary = fh.default_context(), fh.Rotary(frequencies())
    layer, other = (layer_of(fh, m, to_dev(gen.uniform((H,), -2.0, 2.0, 7)), 96, fh.PrefillProjection.I16) for _ in range(2))
    places = lambda first, n: to_dev(np.arange(first, first + n, dtype=np.float32)[:, None] * np.array([[1.0, 0.1, 0.2]], np.float32))  # noqa: E731

    def prompt(layer, n, seed):
        layer.len = 0  # the next prompt
        layer.prefill(to_dev(gen.normal((n, DIM), 1.0, seed)), rotary.at(places(0, n)), 0, 4)

    positions, h = places(20, rows), torch.zeros(rows, DIM, device="cuda:0")
    prompt(layer, 20, 11)
    layer.decode(h.clone(), rotary.at(positions))  # the buffers grow uncaptured
    prompt(layer, 20, 11)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.use_stream(torch.cuda.current_stream())
        layer.decode(h, rotary.at(positions))
    ctx.use_stream(torch.cuda.current_stream())
    kept = []
    for step in range(4):
        x = gen.normal((rows, DIM), 1.0, 31 + step)
        prompt(layer, 60 + step, 41 + step)
        kept.append(torch.full((60 * H * 64,), 1e30, device="cuda:0"))
        prompt(layer, 20, 61 + step)
        h.copy_(to_dev(x))
        graph.replay()
        torch.cuda.synchronize()
        prompt(other, 20, 61 + step)
        want = to_dev(x)
        other.decode(want, rotary.at(positions))
        assert_bitwise(host(h), host(want), f"step {step}")
    assert all((host(t) == np.float32(1e30)).all() for t in kept)
