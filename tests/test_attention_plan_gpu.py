"""What is changed in a plan holds for both ways a call takes: plain tensors
(the C binding) and other views."""
import numpy as np
import pytest
import torch

import vortx_amd as vx
from vortx_amd import _ffi
from tests.helpers import note
from tests.test_attention_gpu import DEV, Q4, Q8, Batch, _gpu

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv():
    assert torch.cuda.is_available()
    return vx.KvAttention(0)


def _view(t):
    return t.flatten(), vx.TensorLayout(tuple(t.shape), tuple(t.stride()), 3)


WAYS = [pytest.param(lambda t: t, id="tensors"), pytest.param(_view, id="views")]


@pytest.fixture
def batch(kv):
    return Batch(kv, np.random.default_rng(21), [3000, 70], [1, 1], 2, 4, 64, 16, (Q8, Q8))


@pytest.mark.parametrize("way", WAYS)
def test_workspace(kv, batch, way):
    note("plan: workspace")
    plan = batch.check(kv)
    want, q, out = batch.out.clone(), _gpu(batch.q), torch.empty_like(batch.out)
    old = plan.workspace
    # another one: it is used, the old one is not
    new = torch.zeros(plan.ws_bytes + 64, dtype=torch.uint8, device=DEV)
    plan.workspace = new
    old.fill_(77)
    kv.attend(out, way(q), plan)
    assert torch.equal(out, want) and (old == 77).all() and new.any()
    # none: the keys are not split
    plan.ws = None
    new.fill_(77)
    kv.attend(out, way(q), plan)
    assert (out - want).abs().max() < 2e-6 and (new == 77).all()
    # a byte short
    plan.workspace = new
    plan.ws_bytes = plan.ws_bytes - 65
    with pytest.raises(vx.VortxError, match="workspace") as e:
        kv.attend(out, way(q), plan)
    assert e.value.status == _ffi.VX_ERR_INVALID


@pytest.mark.parametrize("way", WAYS)
def test_cache_options_and_heads(kv, batch, way):
    note("plan: cache, options, heads")
    plan = batch.check(kv)
    q, out = _gpu(batch.q), torch.empty_like(batch.out)
    other = Batch(kv, np.random.default_rng(21), [3000, 70], [1, 1], 2, 4, 64, 16, (Q8, Q4))
    other.check(kv)
    plan.cache = other.cache
    kv.attend(out, way(q), plan)
    assert torch.equal(out, other.out)
    other.check(kv, window=40)
    plan.opts = _ffi.VxAttnOpts(0.0, 0.0, None, None, None, _ffi.VX_ATTN_CAUSAL, 40)
    kv.attend(out, way(q), plan)
    assert (out - other.out).abs().max() < 2e-6
    plan.q_heads = 4
    with pytest.raises(vx.VortxError, match="heads"):
        kv.attend(out, way(q), plan)
