"""Caps of any size: one that no score comes near changes nothing, one that all
scores are far above leaves no difference between keys."""
import numpy as np
import pytest
import torch

import vortx_amd as vx
from tests.attention_look import attend
from tests.helpers import note
from tests.test_attention_gpu import DEV, Q8, Batch, _gpu

pytestmark = pytest.mark.gpu
ROWS = [(64, 2, 2), (64, 60, 4), (128, 31, 4), (128, 70, 4), (256, 70, 3)]  # 16 rows, 128 and 256 a workgroup


@pytest.fixture(scope="module")
def kv():
    assert torch.cuda.is_available()
    return vx.KvAttention(0)


@pytest.mark.parametrize("cap", [1e-45, 1e-39, 1e-30, 1e-12, 1e6, 1e12, 1e25, 1e36, 3.4e38])
@pytest.mark.parametrize("dim,queries,group", ROWS)
def test_caps_of_any_size(kv, cap, dim, queries, group):
    note(f"cap {cap} {dim} {queries} {group}")
    rng = np.random.default_rng(dim)
    b = Batch(kv, rng, [queries + 60], [queries], 1, group, dim, 16, (Q8, Q8))
    b.q[0] = 0.0  # scores of nothing
    cap = float(np.float32(cap))
    want, tol = attend(b.q, b.kd, b.vd, b.starts, b.lens, softcap=cap)
    out = torch.full(b.q.shape, float("nan"), device=DEV)
    kv.attend(out, _gpu(b.q), b.plan(kv, softcap=cap))
    d = np.abs(out.cpu().numpy() - want)
    assert (d <= tol).all(), f"worst {np.nanmax(d / tol):.3g} of the tolerance"


@pytest.mark.parametrize("dim,queries,group", ROWS[1:4])
def test_scores_past_a_large_cap(kv, dim, queries, group):
    note(f"scores past a large cap {dim} {queries} {group}")
    rng = np.random.default_rng(dim)
    b = Batch(kv, rng, [queries + 60], [queries], 1, group, dim, 16, (Q8, Q8))
    b.q *= np.float32(1e6)
    want, tol = attend(b.q, b.kd, b.vd, b.starts, b.lens, softcap=1e5)
    # scores of 1e6 are off by 1 or so in f32: the keys that count are one or two, and the result is among them
    out = torch.full(b.q.shape, float("nan"), device=DEV)
    kv.attend(out, _gpu(b.q), b.plan(kv, softcap=1e5))
    assert torch.isfinite(out).all() and (np.abs(out.cpu().numpy()) <= np.abs(b.vd[0]).max() * 1.001).all()
