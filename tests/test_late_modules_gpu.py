"""The attention's kernels are loaded at their first use: in a captured graph too."""
import pytest
import torch

import vortx_amd as vx
from tests.helpers import note

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_a_first_call_that_is_captured(dim):
    note(f"first call captured {dim}")
    g = torch.Generator(device=DEV).manual_seed(dim)
    k, v = (torch.randn(5, 2, dim, generator=g, device=DEV) for _ in range(2))
    slots = torch.arange(5, dtype=torch.int32, device=DEV)
    cache = vx.KvCache(2, 16, 2, dim)
    outs = [torch.full((5, 2, dim), float("nan"), device=DEV) for _ in range(4)]
    other = vx.KvAttention(0)
    fresh = vx.KvAttention(0)  # nothing of its attention is loaded
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        fresh.write(cache, k, v, slots)
        fresh.read(outs[0], outs[1], cache, slots)
    for i in range(3):
        k.copy_(torch.randn(k.shape, generator=g, device=DEV))
        outs[0].fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        other.write(cache, k, v, slots)
        other.read(outs[2], outs[3], cache, slots)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3]), i
        assert (outs[0] - k).abs().max() <= k.abs().max() / 200
