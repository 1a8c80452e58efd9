"""Blocks of 32 dims of one key that are far from each other in size: each
comes out as precise as if the others were not there, in every size of kernel."""
import numpy as np
import pytest
import torch

import vortx_amd as vx
from tests.attention_look import attend
from tests.helpers import note
from tests.test_attention_gpu import DEV, Q4, Q8, Batch, _gpu, _normal, _tree, _words

pytestmark = pytest.mark.gpu
ROWS = [(64, 2, 2), (64, 60, 4), (128, 2, 4), (128, 31, 4), (128, 70, 4), (96, 60, 4), (256, 3, 2), (256, 70, 3)]
# largest values of the large and of the small blocks
SIZES = [(300.0, 0.01), (1e4, 1e-3), (1e6, 1.0), (6.0, 1e-2), (6e4, 1e-4)]


@pytest.fixture(scope="module")
def kv():
    assert torch.cuda.is_available()
    return vx.KvAttention(0)


def _check(kv, b, trees=None, **options):
    want, tol = attend(b.q, b.kd, b.vd, b.starts, b.lens, trees=trees, **options)
    plan = b.plan(kv, **options)
    q = _gpu(b.q)
    view = (q.flatten(), vx.TensorLayout(tuple(q.shape), tuple(q.stride()), 3))
    for ws in (True, False):
        if not ws:
            plan.ws = None
        out = torch.full(q.shape, float("nan"), device=DEV)
        if trees is None:
            kv.attend(out, view, plan)
        else:
            kv.attend_tree(out, view, plan, _words(trees))
        d = np.abs(out.cpu().numpy() - want)
        assert (d <= tol).all(), f"worst {np.nanmax(d / tol):.3g} of the tolerance (workspace {ws})"


def _scaled(rng, n, dim, large, small, which):
    """Keys whose first block is `large` and whose others are `small`; which: every key, some, or one of 32."""
    large, small = large / 16, small / 16  # (4 bits: a scale of the largest value / 8 is an f16)
    x = _normal(rng, n, 1, dim) * np.float32(small)
    on = {"every": np.ones(n, bool), "some": rng.random(n) < 0.5, "few": np.arange(n) % 32 == 21}[which]
    x[on, :, :32] *= np.float32(large / small)
    return x.astype(np.float32)


@pytest.mark.parametrize("types", [(Q8, Q8), (Q4, Q4), (Q4, Q8)], ids=["k8v8", "k4v4", "k4v8"])
@pytest.mark.parametrize("which", ["every", "some", "few"])
@pytest.mark.parametrize("large,small", SIZES)
@pytest.mark.parametrize("dim,queries,group", ROWS)
def test_values(kv, types, which, large, small, dim, queries, group):
    note(f"block sizes of values {types} {which} {large} {small} {dim} {queries} {group}")
    rng = np.random.default_rng(dim + queries)
    L = queries + 75
    v = [_scaled(rng, L, dim, large, small, which)]
    _check(kv, Batch(kv, rng, [L], [queries], 1, group, dim, 16, types, v=v))


@pytest.mark.parametrize("types", [(Q8, Q8), (Q4, Q4), (Q8, Q4)], ids=["k8v8", "k4v4", "k8v4"])
@pytest.mark.parametrize("which", ["every", "some", "few"])
@pytest.mark.parametrize("large,small", SIZES)
@pytest.mark.parametrize("dim,queries,group", ROWS)
@pytest.mark.parametrize("beside", [0.0, 1.0], ids=["unasked", "asked"])
def test_keys(kv, types, which, large, small, dim, queries, group, beside):
    """Queries that are nothing in the large block, or so small there that both count."""
    note(f"block sizes of keys {types} {which} {large} {small} {dim} {queries} {group} {beside}")
    rng = np.random.default_rng(dim + queries)
    L = queries + 75
    k = [_scaled(rng, L, dim, large, small, which)]
    b = Batch(kv, rng, [L], [queries], 1, group, dim, 16, types, k=k)
    ratio = max(small / large, 2.0 ** -16) * beside  # (q has 22 bits down to 2^-17 of its row's largest)
    b.q *= np.float32(16 / small)
    b.q[..., :32] *= np.float32(ratio)
    _check(kv, b)


@pytest.mark.parametrize("dim,queries,group", ROWS)
def test_both_with_a_tree_and_options(kv, dim, queries, group):
    note(f"block sizes of both {dim} {queries} {group}")
    rng = np.random.default_rng(dim)
    L = queries + 75
    k, v = [_scaled(rng, L, dim, 1e4, 0.1, "some")], [_scaled(rng, L, dim, 1e4, 0.1, "some")]
    b = Batch(kv, rng, [L], [queries], 1, group, dim, 16, (Q8, Q8), k=k, v=v)
    b.q[..., :32] *= np.float32(1e-4)
    slopes = rng.uniform(0.01, 0.1, b.q_heads).astype(np.float32)
    _check(kv, b, window=50, slopes=slopes, softcap=3.0)
    _check(kv, b, trees=[_tree(rng, queries)], slopes=slopes, first=np.full(queries, 9))


@pytest.mark.parametrize("dim,queries,group", ROWS)
def test_blocks_of_neighbouring_keys(kv, dim, queries, group):
    """One key's first block and another's last are the large ones, each seen by some rows only."""
    note(f"block sizes of neighbours {dim} {queries} {group}")
    rng = np.random.default_rng(dim)
    L = queries + 75
    v = _normal(rng, L, 1, dim) * np.float32(0.01)
    v[::3, :, :32] *= np.float32(1e5)
    v[1::3, :, -32:] *= np.float32(1e5)
    v[L - queries::2] *= np.float32(3e-4)
    b = Batch(kv, rng, [L], [queries], 1, group, dim, 16, (Q8, Q8), v=[v])
    _check(kv, b, first=rng.integers(0, L - 2, queries))
    _check(kv, b, window=2)
