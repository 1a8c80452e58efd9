"""Lengths past max_len or past the page table hide keys and move nothing, and
a tree may have more drafts than its sequence has keys."""
import numpy as np
import pytest
import torch

import vortx_amd as vx
from tests.attention_look import attend
from tests.helpers import note
from tests.test_attention_gpu import DEV, Q4, Q8, Batch, _gpu, _i32, _tree, _words

pytestmark = pytest.mark.gpu
ROWS = [(64, 2, 2), (64, 60, 4), (128, 31, 4), (128, 70, 4), (256, 70, 3)]  # 16 rows, 128 and 256 a workgroup


@pytest.fixture(scope="module")
def kv():
    assert torch.cuda.is_available()
    return vx.KvAttention(0)


def _check(kv, b, max_len, most, trees=None, words=None, cols=None, **options):
    want, tol = attend(b.q, b.kd, b.vd, b.starts, b.lens, trees=trees, most=most, **options)
    options = dict(options)
    if "first" in options:
        options["first"] = _i32(options["first"])
    if "slopes" in options:
        options["slopes"] = _gpu(options["slopes"])
    if "prefix" in options:
        options["prefix"] = _i32(options["prefix"])
    table = b.table if cols is None else b.table[:, :cols]
    plan = kv.plan(b.cache, _i32(table), _i32(b.lens), _i32(b.starts), q_heads=b.q_heads, max_queries=max(b.n), max_len=max_len, **options)
    q = _gpu(b.q)
    view = (q.flatten(), vx.TensorLayout(tuple(q.shape), tuple(q.stride()), 3))
    for ws in (True, False):
        if not ws:
            plan.ws = None
        out = torch.full(q.shape, float("nan"), device=DEV)
        if trees is None:
            kv.attend(out, view, plan)
        else:
            kv.attend_tree(out, view, plan, _words(trees) if words is None else words)
        d = np.abs(out.cpu().numpy() - want)
        assert (d <= tol).all(), f"worst {np.nanmax(d / np.maximum(tol, 1e-30)):.3g} of the tolerance (workspace {ws})"


@pytest.mark.parametrize("dim,queries,group", ROWS)
@pytest.mark.parametrize("cut", [1, 33, 100])
def test_keys_past_the_most(kv, dim, queries, group, cut):
    note(f"past max_len {dim} {queries} {group} {cut}")
    rng = np.random.default_rng(dim + cut)
    lens = [queries + 131, queries + 40]
    b = Batch(kv, rng, lens, [queries] * 2, 1, group, dim, 16, (Q8, Q4))
    most = max(lens) - cut
    slopes = rng.uniform(0.01, 0.3, group).astype(np.float32)
    for options in (dict(), dict(causal=False), dict(slopes=slopes), dict(window=37, slopes=slopes), dict(prefix=[200, 90]),
                    dict(first=rng.integers(0, 100, b.T))):
        _check(kv, b, most, most, **options)
    _check(kv, b, most, most, trees=[_tree(rng, queries) for _ in range(2)], slopes=slopes)
    _check(kv, b, most, most, trees=[_tree(rng, queries) for _ in range(2)], window=37)


@pytest.mark.parametrize("dim,queries,group", ROWS)
def test_keys_past_the_page_table(kv, dim, queries, group):
    note(f"past the table {dim} {queries} {group}")
    rng = np.random.default_rng(dim)
    lens = [queries + 131, queries + 40]
    b = Batch(kv, rng, lens, [queries] * 2, 1, group, dim, 16, (Q8, Q8))
    cols = (queries + 100) // 16
    slopes = rng.uniform(0.01, 0.3, group).astype(np.float32)
    _check(kv, b, max(lens), 16 * cols, cols=cols, slopes=slopes)
    _check(kv, b, max(lens), 16 * cols, cols=cols, trees=[_tree(rng, queries) for _ in range(2)], slopes=slopes)


@pytest.mark.parametrize("dim,queries,group", ROWS)
@pytest.mark.parametrize("short", [1, 2, 40])
def test_more_drafts_than_keys(kv, dim, queries, group, short):
    """The drafts' keys are the last ones: those that would lie before the first do not exist."""
    note(f"more drafts than keys {dim} {queries} {group} {short}")
    rng = np.random.default_rng(dim + short)
    L = max(queries - short, 1)
    b = Batch(kv, rng, [L, 50], [queries, 1], 1, group, dim, 16, (Q8, Q8))
    slopes = rng.uniform(0.01, 0.3, group).astype(np.float32)
    trees = [rng.random((queries, queries)) < 0.4, np.ones((1, 1), bool)]
    _check(kv, b, 500, 500, trees=trees)
    _check(kv, b, 500, 500, trees=trees, slopes=slopes)
    _check(kv, b, 500, 500, trees=trees, window=9)
