"""Pages, rotation and 8-bit products: their kernels are loaded at their first use, in a
captured graph too."""
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
kv, i8 = vx.KvAttention(0), vx.Int8Gemm(0)
g = torch.Generator(device=DEV).manual_seed(1)
x, w, how = torch.randn(6, 128, generator=g, device=DEV), torch.randn(32, 128, generator=g, device=DEV), kv.rotation(vx.rotation_freqs(64))
rows, outs = vx.Int8Rows.empty(32, 128), [torch.zeros(6, 32, device=DEV) for _ in range(2)]
pages, step, want = vx.KvPages(8, 16, 2, 4), vx.KvStep(2, 6), torch.tensor([5, 1], dtype=torch.int32, device=DEV)
zero, ws, y = torch.zeros(2, dtype=torch.int32, device=DEV), i8.workspace(6, 128), torch.zeros(6, 2, 64, device=DEV)

def run(out):
    kv.resize(pages, want, step)  # the process's first calls are captured
    kv.rotate(y, x.unflatten(1, (2, 64)), None, None, step.positions, how)
    i8.quantize(rows, w)
    i8.dispatch(out, y.flatten(1), rows, workspace=ws)

stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
    run(outs[0])
for i in range(3):
    x.copy_(torch.randn(x.shape, generator=g, device=DEV))
    w.copy_(torch.randn(w.shape, generator=g, device=DEV))
    outs[0].zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert step.positions.tolist() == [0, 1, 2, 3, 4, 0] and pages.lens.tolist() == [5, 1]
    kv.resize(pages, zero, step)
    run(outs[1])
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1]) and outs[0].abs().max() > 1, i
    kv.resize(pages, zero, step)
    print(i, "fine", flush=True)
"""


def test_first_calls_that_are_captured():
    note("first calls captured (a process of their own: the kernels are loaded once in one)")
    r = subprocess.run([sys.executable, "-c", CHILD], cwd=ROOT, capture_output=True, text=True, timeout=90)
    assert r.returncode == 0 and r.stdout.count("fine") == 3, (r.stdout + r.stderr)[-3000:]
