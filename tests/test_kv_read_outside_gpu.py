"""Reading slots outside the cache: zeros, also where whole groups of four
consecutive slots lie past its end (calls of many tokens go by such groups)."""
import numpy as np
import pytest
import torch

import vortx_amd as vx
from tests import attention_oracle as A
from tests.helpers import note

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.fixture(scope="module")
def kv():
    assert torch.cuda.is_available()
    return vx.KvAttention(0)


def _gpu(a):
    return torch.tensor(np.ascontiguousarray(a), device=DEV)


@pytest.mark.parametrize("types", [(vx.VX_Q8_0, vx.VX_Q4_0), (vx.VX_Q4_0, vx.VX_Q8_0)], ids=["k8v4", "k4v8"])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("first", [200, 201, 203, 508, 600])
@pytest.mark.parametrize("strided", [False, True], ids=["rows", "strided"])
def test_consecutive_slots_past_the_last_page_read_as_zeros(kv, types, dim, first, strided):
    note(f"past the end {types} {dim} {first} {strided}")
    rng = np.random.default_rng(first)
    heads, pages, page = 2, 16, 32
    cache = vx.KvCache(pages, page, heads, dim, *types)
    n = pages * page
    k, v = (rng.standard_normal((n, heads, dim)).astype(np.float32) for _ in range(2))
    kv.write(cache, _gpu(k), _gpu(v), _gpu(np.arange(n, dtype=np.int32)))
    slots = np.arange(first, first + 403, dtype=np.int32)
    inside = slots < n
    want = [np.zeros((403, heads, dim), np.float32) for _ in range(2)]
    for w, x, t in zip(want, (k, v), types):
        w[inside] = A.values(x[slots[inside]], t)
    if strided:
        outs = [torch.full((403, heads, dim + 1), float("nan"), device=DEV)[..., :dim] for _ in range(2)]
    else:
        outs = [torch.full((403, heads, dim), float("nan"), device=DEV) for _ in range(2)]
    kv.read(*outs, cache, _gpu(slots))
    for got, w in zip(outs, want):
        assert np.array_equal(got.cpu().numpy(), w)
    for i in range(2):  # one of the two alone
        only = [None, None]
        only[i] = torch.full((403, heads, dim), float("nan"), device=DEV)
        kv.read(*only, cache, _gpu(slots))
        assert np.array_equal(only[i].cpu().numpy(), want[i])


def test_a_cache_without_pages_reads_as_zeros(kv):
    cache = vx.KvCache(0, 16, 2, 64)
    for first in (0, 1):
        outs = [torch.full((300, 2, 64), float("nan"), device=DEV) for _ in range(2)]
        kv.read(*outs, cache, _gpu(np.arange(first, first + 300, dtype=np.int32)))
        assert all((o == 0).all() for o in outs)
