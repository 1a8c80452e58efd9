"""The attention's kernels are loaded at their first use: in a captured graph too."""
import os
import subprocess
import sys

import pytest

from tests.helpers import note

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = """
import torch
import vortx_amd as vx
DEV = torch.device("cuda:0")
for dim in (64, 96, 128, 256):
    g = torch.Generator(device=DEV).manual_seed(dim)
    k, v = (torch.randn(5, 2, dim, generator=g, device=DEV) for _ in range(2))
    slots = torch.arange(5, dtype=torch.int32, device=DEV)
    cache, kv = vx.KvCache(2, 16, 2, dim), vx.KvAttention(0)
    outs = [torch.full((5, 2, dim), float("nan"), device=DEV) for _ in range(4)]
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        kv.write(cache, k, v, slots)  # the process's first call of this head size
        kv.read(outs[0], outs[1], cache, slots)
    for i in range(3):
        k.copy_(torch.randn(k.shape, generator=g, device=DEV))
        outs[0].fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        kv.write(cache, k, v, slots)
        kv.read(outs[2], outs[3], cache, slots)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3]), (dim, i)
        assert (outs[0] - k).abs().max() <= k.abs().max() / 200, (dim, i)
    print(dim, "fine", flush=True)
"""


def test_first_calls_that_are_captured():
    note("first calls captured (a process of their own: the kernels are loaded once in one)")
    r = subprocess.run([sys.executable, "-c", CHILD], cwd=ROOT, capture_output=True, text=True, timeout=90)
    assert r.returncode == 0 and r.stdout.count("fine") == 4, (r.stdout + r.stderr)[-3000:]
