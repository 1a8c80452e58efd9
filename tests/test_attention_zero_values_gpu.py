"""Keys whose values are all zeros beside a neighbour that no row sees, of
any size or never written: their weights cost the others no precision."""
import numpy as np
import pytest
import torch

import vortx_amd as vx
from tests.helpers import note
from tests.test_attention_block_sizes_gpu import ROWS, _check
from tests.test_attention_gpu import Q4, Q8, Batch, _normal
from tests.test_attention_unwritten_gpu import Unwritten

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv():
    assert torch.cuda.is_available()
    return vx.KvAttention(0)


@pytest.mark.parametrize("types", [(Q8, Q8), (Q4, Q4)], ids=["k8v8", "k4v4"])
@pytest.mark.parametrize("dim,queries,group", ROWS)
@pytest.mark.parametrize("beside", ["huge", "huge_tokens", 0x1F, "random"])
def test_zeros_beside_what_no_row_sees(kv, types, dim, queries, group, beside):
    note(f"zeros beside {beside} {types} {dim} {queries} {group}")
    rng = np.random.default_rng(dim + queries)
    first, L = 43, 43 + max(queries, 30)  # the last of its four keys
    k, v = _normal(rng, L, 1, dim) * np.float32(0.1), _normal(rng, L, 1, dim)
    v[first] = 0.0
    v[first + 5] = 0.0
    if isinstance(beside, str) and beside.startswith("huge"):
        v[:first] *= np.float32(1e6)
        b = Batch(kv, rng, [L], [queries], 1, group, dim, 16, types, k=[k], v=[v])
    else:
        b = Batch(Unwritten(kv, beside, types, [first], rng), rng, [L], [queries], 1, group, dim, 16, types, k=[k], v=[v])
    _check(kv, b, first=np.full(queries, first))
    if beside == "huge_tokens":  # many tokens at once are written by fours
        again = [_normal(rng, 300, 1, dim) * np.float32(0.1), _normal(rng, 300, 1, dim)]
        again[1][150] *= np.float32(1e6)
        again[1][151] = 0.0
        b = Batch(kv, rng, [300], [queries], 1, group, dim, 16, types, k=[again[0]], v=[again[1]])
        _check(kv, b, first=np.full(queries, 151))
