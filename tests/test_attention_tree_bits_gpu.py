"""Bits of a tree's rows beyond a sequence's drafts stand for nothing."""
import numpy as np
import pytest
import torch

import vortx_amd as vx
from tests.helpers import note
from tests.test_attention_gpu import DEV, Q8, Batch, _gpu, _tree
from tests.test_attention_lengths_gpu import ROWS, _check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv():
    assert torch.cuda.is_available()
    return vx.KvAttention(0)


@pytest.mark.parametrize("dim,queries,group", ROWS)
def test_bits_past_the_drafts_stand_for_nothing(kv, dim, queries, group):
    """Sequences of a batch have trees of different sizes in rows of the same length: a draft's
    position counts the drafts that there are."""
    note(f"bits past the drafts {dim} {queries} {group}")
    rng = np.random.default_rng(dim)
    n = [queries, max(queries - 7, 1)]
    b = Batch(kv, rng, [queries + 60, queries + 30], n, 1, group, dim, 16, (Q8, Q8))
    trees = [_tree(rng, i) for i in n]
    words = -(-queries // 32) + 1
    rows = []
    for t in trees:
        m = rng.random((t.shape[0], 32 * words)) < 0.5
        m[:, :t.shape[1]] = t
        rows.append(np.packbits(m, axis=1, bitorder="little").view(np.int32))
    slopes = rng.uniform(0.01, 0.3, group).astype(np.float32)
    words = torch.tensor(np.concatenate(rows), device=DEV)
    _check(kv, b, 500, 500, trees=trees, words=words, slopes=slopes)
    _check(kv, b, 500, 500, trees=trees, words=words, window=11)
