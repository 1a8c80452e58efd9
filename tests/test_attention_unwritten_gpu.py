"""Slots that were never written, in pages of any contents: no row sees them,
and what they hold reaches no result. In every size of kernel (16, 128 and 256
query rows, keys dealt out or not)."""
import numpy as np
import pytest
import torch

import vortx_amd as vx
from tests.helpers import note
from tests.test_attention_gpu import DEV, Q4, Q8, Batch, _gpu, _i32, _tree, _words

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv():
    assert torch.cuda.is_available()
    return vx.KvAttention(0)


def _fill(cache, kind, types, rng):
    """Bytes of a cache before anything is written."""
    per = sum(16 * (cache.dim // 32) * (34 if t == Q8 else 18) for t in types) + 32  # a record; its sizes are the last 32 bytes
    data = cache.data
    if isinstance(kind, int):
        data.fill_(kind)
    elif kind == "random":
        data.copy_(torch.tensor(rng.integers(0, 256, data.numel(), dtype=np.uint8)))
    else:  # scales (and all else) of one f16, sizes of one value
        scale, size = kind
        data.view(torch.float16).fill_(scale)
        data[:data.numel() // per * per].view(-1, per)[:, -32:] = size


class Unwritten:
    """Stands in for KvAttention where a Batch writes: `begin[s]` keys of sequence s stay as they are."""

    def __init__(self, kv, kind, types, begin, rng):
        self.kv, self.kind, self.types, self.begin, self.rng = kv, kind, types, list(begin), rng

    def write(self, cache, k, v, slots):
        if self.kind is not None:
            _fill(cache, self.kind, self.types, self.rng)
            self.kind = None
        b = self.begin.pop(0)
        if b < k.shape[0]:
            self.kv.write(cache, k[b:], v[b:], slots[b:])


FILLS = [0x7F, 0xC8, 0x96, 0x1F, 0xFE, "random", (3.0, 0), (float("nan"), 127), (float("inf"), 17), (60000.0, 16), (float("nan"), 1)]
IDS = ["7f", "c8", "96", "1f", "fe", "random", "size_0", "nan_127", "inf_17", "large_16", "nan_1"]
# dim, query tokens, query heads for each: 16 rows, 128 and 256 a workgroup
ROWS = [(64, 2, 2), (64, 60, 4), (128, 31, 4), (128, 70, 4), (96, 60, 4), (256, 70, 3)]


def _both(b, kv, **options):
    """With a workspace (the keys dealt out) and without."""
    plan = b.check(kv, **options)
    trees = options.pop("trees", None)
    got = b.out.clone()
    plan.ws = None
    out, q = torch.full(b.q.shape, float("nan"), device=DEV), _gpu(b.q)
    view = (q.flatten(), vx.TensorLayout(tuple(q.shape), tuple(q.stride()), 3))
    if trees is None:
        kv.attend(out, view, plan)
    else:
        kv.attend_tree(out, view, plan, _words(trees))
    assert torch.isfinite(out).all()
    assert (out - got).abs().max() <= 4e-6 * max(1.0, got.abs().max().item())


@pytest.mark.parametrize("kind", FILLS, ids=IDS)
@pytest.mark.parametrize("dim,queries,group", ROWS)
@pytest.mark.parametrize("types", [(Q8, Q8), (Q4, Q8), (Q8, Q4)], ids=["k8v8", "k4v8", "k8v4"])
def test_keys_before_the_first(kv, kind, dim, queries, group, types):
    note(f"unwritten before the first {kind} {dim} {queries} {group} {types}")
    rng = np.random.default_rng(dim)
    lens = [queries + 90, queries + 40]
    begin = [5, 21]
    b = Batch(Unwritten(kv, kind, types, begin, rng), rng, lens, [queries] * 2, 1, group, dim, 16, types)
    first = np.repeat(begin, queries)
    _both(b, kv, first=first)
    _both(b, kv, first=first, causal=False)
    _both(b, kv, trees=[_tree(rng, queries) for _ in range(2)], first=first)


@pytest.mark.parametrize("kind", FILLS, ids=IDS)
@pytest.mark.parametrize("dim,queries,group", ROWS)
def test_keys_before_the_window_and_pages_that_are_gone(kv, kind, dim, queries, group):
    note(f"unwritten before the window {kind} {dim} {queries} {group}")
    rng = np.random.default_rng(dim + 1)
    types, window = (Q8, Q8), 30
    lens = [queries + 101, queries + 33]
    begin = [L - queries - window + 1 for L in lens]
    b = Batch(Unwritten(kv, kind, types, begin, rng), rng, lens, [queries] * 2, 1, group, dim, 16, types)
    for s, at in enumerate(begin):  # their pages went back
        b.table[s, :at // 16] = -1
    _both(b, kv, window=window)
