"""The quantized key/value cache and the attention over it against plain
restatements in 64 bits (tests/attention_oracle.py)."""
import numpy as np
import pytest
import torch

import vortx_amd as vx
from tests import attention_oracle as A
from tests.helpers import note
from vortx_amd import _ffi

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
Q8, Q4 = vx.VX_Q8_0, vx.VX_Q4_0
TYPES = [(Q8, Q8), (Q8, Q4), (Q4, Q8), (Q4, Q4)]


@pytest.fixture(scope="module")
def kv():
    assert torch.cuda.is_available()
    return vx.KvAttention(0)


def _i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)


def _gpu(a):
    return torch.tensor(np.ascontiguousarray(a), dtype=torch.float32, device=DEV)


def _normal(rng, *shape):
    return rng.standard_normal(shape).astype(np.float32)


class Batch:
    """Sequences in a cache whose other bytes are all ones (NaN scales)."""

    def __init__(self, kv, rng, lens, queries, heads, group, dim, page, types, k=None, v=None, spare=3):
        self.lens, self.n = list(lens), list(queries)
        self.starts = np.concatenate([[0], np.cumsum(self.n)]).astype(np.int32)
        self.T = int(self.starts[-1])
        need = [-(-L // page) for L in self.lens]
        pages, cols = sum(need) + spare, max(max(need), 1)
        order = rng.permutation(pages)
        self.table = np.full((len(self.lens), cols), 2 ** 31 - 1, np.int32)  # entries past the end: no page
        at = 0
        for s, c in enumerate(need):
            self.table[s, :c] = order[at:at + c]
            at += c
        self.cache = vx.KvCache(pages, page, heads, dim, *types)
        self.cache.data.fill_(255)
        self.k = k if k is not None else [_normal(rng, L, heads, dim) for L in self.lens]
        self.v = v if v is not None else [_normal(rng, L, heads, dim) for L in self.lens]
        for s, L in enumerate(self.lens):
            if L:
                kv.write(self.cache, _gpu(self.k[s]), _gpu(self.v[s]), _i32(self.slots(s, np.arange(L))))
        self.kd = [A.values(x, types[0]) for x in self.k]
        self.vd = [A.values(x, types[1]) for x in self.v]
        self.q = _normal(rng, self.T, heads * group, dim)
        self.q_heads = heads * group

    def slots(self, s, pos):
        p = self.cache.page_tokens
        return self.table[s, pos // p].astype(np.int64) * p + pos % p

    def plan(self, kv, **options):
        for name in ("first", "prefix"):
            if options.get(name) is not None:
                options[name] = _i32(options[name])
        if options.get("slopes") is not None:
            options["slopes"] = _gpu(options["slopes"])
        return kv.plan(self.cache, _i32(self.table), _i32(self.lens), _i32(self.starts), q_heads=self.q_heads,
                       max_queries=max(max(self.n), 1), max_len=max(max(self.lens), 1), **options)

    def check(self, kv, trees=None, q=None, **options):
        q = self.q if q is None else q
        want, tol = A.attend(q, self.kd, self.vd, self.starts, self.lens, trees=trees, **options)
        plan = self.plan(kv, **options)
        gq, out = _gpu(q), torch.full(q.shape, float("nan"), device=DEV)
        if trees is None:
            kv.attend(out, gq, plan)
        else:
            kv.attend_tree(out, gq, plan, _words(trees))
        torch.cuda.synchronize()
        got = out.cpu().numpy().astype(np.float64)
        self.out = out
        assert np.array_equal(np.isnan(got), np.isnan(want))
        d = np.abs(got - want)
        bad = d > tol
        assert not bad.any(), f"{int(bad.sum())} of {bad.size} off, worst {np.nanmax(d / np.maximum(tol, 1e-300)):.3g} of the tolerance"
        return plan


def _words(trees):
    words = max(1, -(-max(t.shape[0] for t in trees) // 32))
    rows = []
    for t in trees:
        m = np.zeros((t.shape[0], 32 * words), bool)
        m[:, :t.shape[1]] = t
        rows.append(np.packbits(m, axis=1, bitorder="little").view(np.int32))
    return torch.tensor(np.concatenate(rows), device=DEV)


def _tree(rng, n, reach=5):
    t = np.eye(n, dtype=bool)
    for j in range(n):
        p = int(rng.integers(max(-1, j - reach), j)) if j else -1
        if p >= 0:
            t[j] |= t[p]
    return t


# ------------------------------------------------------- rows in and out
def _edge_rows(rng, T, heads, dim):
    """Rows with blocks where a quantizer can go wrong."""
    x = _normal(rng, T, heads, dim) * np.exp(rng.uniform(-8, 8, (T, heads, 1))).astype(np.float32)
    f = x.reshape(T * heads, -1, 32)
    f[0, 0] = 0.0
    f[1 % len(f), 0] = -0.0
    f[2 % len(f), 0] = 1e-9             # the scale underflows to a subnormal
    f[3 % len(f), 0] = 1e-12            # the scale underflows to zero
    f[4 % len(f), 0, :2] = [3.0, -3.0]  # a tie of magnitudes
    f[4 % len(f), 0, 2:] = np.linspace(-3, 3, 30)
    f[5 % len(f), 0] = np.arange(32) * 0.5 - 8  # halves
    f[6 % len(f), 1] = 1e5
    return x


@pytest.mark.parametrize("types", TYPES, ids=["k8v8", "k8v4", "k4v8", "k4v4"])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("T,heads,page", [(1, 1, 16), (7, 3, 32), (70, 2, 16), (129, 5, 64)])
def test_rows_come_back_as_the_blocks_values(kv, types, dim, T, heads, page):
    note(f"rows {types} {dim} {T} {heads} {page}")
    rng = np.random.default_rng(T * dim)
    cache = vx.KvCache(-(-T // page) + 2, page, heads, dim, *types)
    k, v = _edge_rows(rng, T, heads, dim), _edge_rows(rng, T, heads, dim)[::-1].copy()
    slots = _i32(rng.permutation(cache.pages * page)[:T])
    kv.write(cache, _gpu(k), _gpu(v), slots)
    ko, vo = (torch.full((T, heads, dim), float("nan"), device=DEV) for _ in range(2))
    kv.read(ko, vo, cache, slots)
    assert np.array_equal(ko.cpu().numpy(), A.values(k, types[0]).astype(np.float32))
    assert np.array_equal(vo.cpu().numpy(), A.values(v, types[1]).astype(np.float32))


@pytest.mark.parametrize("types", [(Q8, Q4), (Q4, Q8)], ids=["k8v4", "k4v8"])
def test_rows_in_order_fill_pages(kv, types):
    """Consecutive slots, any first slot and any count: what a prompt writes."""
    rng = np.random.default_rng(3)
    for first, T in [(0, 64), (3, 61), (13, 1), (15, 2), (16, 33), (5, 100)]:
        cache = vx.KvCache(8, 16, 2, 128, *types)
        cache.data.fill_(255)
        k, v = _normal(rng, T, 2, 128), _normal(rng, T, 2, 128)
        slots = _i32(np.arange(first, first + T))
        kv.write(cache, _gpu(k), _gpu(v), slots)
        ko, vo = torch.empty(T, 2, 128, device=DEV), torch.empty(T, 2, 128, device=DEV)
        kv.read(ko, vo, cache, slots)
        assert np.array_equal(ko.cpu().numpy(), A.values(k, types[0]).astype(np.float32)), (first, T)
        assert np.array_equal(vo.cpu().numpy(), A.values(v, types[1]).astype(np.float32)), (first, T)


@pytest.mark.parametrize("types", TYPES, ids=["k8v8", "k8v4", "k4v8", "k4v4"])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("kind", ["aligned", "off_by_one", "off_by_three", "sequences", "shuffled", "gaps"])
def test_many_rows(kv, types, dim, kind):
    """Enough tokens to go by fours: runs of slots that begin anywhere, end in a
    group of four, are broken, or none."""
    note(f"many rows {types} {dim} {kind}")
    rng = np.random.default_rng(dim)
    T, heads = 403, 3
    slots = {"aligned": np.arange(T), "off_by_one": np.arange(1, T + 1), "off_by_three": np.arange(3, T + 3),
             "sequences": np.concatenate([np.arange(0, 130), np.arange(146, 146 + 131), np.arange(301, 301 + 142)]),
             "shuffled": rng.permutation(512)[:T], "gaps": np.arange(T) + np.arange(T) // 7}[kind]
    outside = rng.choice(T, 9, replace=False) if kind in ("gaps", "sequences") else []
    slots[outside] = rng.choice([-1, -8, 512, 2 ** 31 - 4], len(outside))
    cache = vx.KvCache(16, 32, heads, dim, *types)
    cache.data.fill_(255)
    k, v = _edge_rows(rng, T, heads, dim), _edge_rows(rng, T, heads, dim)
    kv.write(cache, _gpu(k), _gpu(v), _i32(slots))
    ko, vo = (torch.full((T, heads, dim), float("nan"), device=DEV) for _ in range(2))
    kv.read(ko, vo, cache, _i32(slots))
    wk, wv = A.values(k, types[0]).astype(np.float32), A.values(v, types[1]).astype(np.float32)
    wk[outside], wv[outside] = 0, 0
    assert np.array_equal(ko.cpu().numpy(), wk) and np.array_equal(vo.cpu().numpy(), wv)
    # attention reads what was written, sizes of the scales among it
    inside = slots[(slots >= 0) & (slots < 512)]
    other = vx.KvCache(16, 32, heads, dim, *types)
    other.data.fill_(255)
    for i in np.argsort(rng.random(T))[:]:
        if 0 <= slots[i] < 512 and i % 97 == 0:  # some, one by one
            kv.write(other, _gpu(k[i:i + 1]), _gpu(v[i:i + 1]), _i32(slots[i:i + 1]))
            at = int(slots[i])
            one = [kv.plan(c, _i32([[at // 32]]), _i32([at % 32 + 1]), _i32([0, 1]), q_heads=heads, max_queries=1, max_len=32,
                           first=_i32([at % 32])) for c in (cache, other)]
            q, outs = _gpu(_normal(rng, 1, heads, dim)), [torch.empty(1, heads, dim, device=DEV) for _ in range(2)]
            for plan, out in zip(one, outs):
                kv.attend(out, q, plan)
            assert torch.equal(outs[0], outs[1])
    assert len(inside) >= T - 9


@pytest.mark.parametrize("types", TYPES, ids=["k8v8", "k8v4", "k4v8", "k4v4"])
def test_writing_a_slot_leaves_the_others(kv, types):
    rng = np.random.default_rng(5)
    cache = vx.KvCache(3, 16, 2, 96, *types)
    n = 48
    k, v = _normal(rng, n, 2, 96), _normal(rng, n, 2, 96)
    kv.write(cache, _gpu(k), _gpu(v), _i32(np.arange(n)))
    for slot in (0, 3, 17, 47):
        k[slot], v[slot] = _normal(rng, 2, 96), _normal(rng, 2, 96)
        kv.write(cache, _gpu(k[slot:slot + 1]), _gpu(v[slot:slot + 1]), _i32([slot]))
    # slots outside the cache: left out
    out = _normal(rng, 4, 2, 96)
    kv.write(cache, _gpu(out), _gpu(out), _i32([-1, 48, 2 ** 31 - 1, -2 ** 31]))
    ko, vo = torch.empty(n + 2, 2, 96, device=DEV), torch.empty(n + 2, 2, 96, device=DEV)
    kv.read(ko, vo, cache, _i32(list(range(n)) + [-1, 48]))
    zeros = np.zeros((2, 2, 96))
    assert np.array_equal(ko.cpu().numpy(), np.concatenate([A.values(k, types[0]), zeros]).astype(np.float32))
    assert np.array_equal(vo.cpu().numpy(), np.concatenate([A.values(v, types[1]), zeros]).astype(np.float32))


@pytest.mark.parametrize("types", TYPES, ids=["k8v8", "k8v4", "k4v8", "k4v4"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 1e8, -3e38])
def test_blocks_that_a_scale_cannot_hold_read_as_nan(kv, types, bad):
    rng = np.random.default_rng(6)
    cache = vx.KvCache(1, 16, 1, 64, *types)
    k, v = _normal(rng, 2, 1, 64), _normal(rng, 2, 1, 64)
    k[0, 0, 40] = bad
    v[1, 0, 3] = bad
    kv.write(cache, _gpu(k), _gpu(v), _i32([4, 5]))
    ko, vo = torch.empty(2, 1, 64, device=DEV), torch.empty(2, 1, 64, device=DEV)
    kv.read(ko, vo, cache, _i32([4, 5]))
    want_k, want_v = np.zeros((2, 1, 64), bool), np.zeros((2, 1, 64), bool)
    want_k[0, 0, 32:], want_v[1, 0, :32] = True, True
    assert np.array_equal(np.isnan(ko.cpu().numpy()), want_k) and np.array_equal(np.isnan(vo.cpu().numpy()), want_v)
    assert np.array_equal(ko[1].cpu().numpy(), A.values(k[1], types[0]).astype(np.float32))


def test_rows_of_any_strides(kv):
    rng = np.random.default_rng(7)
    T, H, D = 21, 3, 64
    cache = vx.KvCache(4, 16, H, D, Q8, Q4)
    slots = _i32(rng.permutation(64)[:T])
    k, v = _normal(rng, T, H, D), _normal(rng, T, H, D)
    wide = torch.zeros(T, H, D + 3, device=DEV)  # rows that are not 16-byte aligned
    wide[..., 1:D + 1] = _gpu(k)
    kv.write(cache, wide[..., 1:D + 1], _gpu(v).permute(1, 2, 0).contiguous().permute(2, 0, 1), slots)
    ko = torch.zeros(H, T, 2 * D, device=DEV).permute(1, 0, 2)[..., ::2]
    vo = torch.zeros(D, H, T, device=DEV).permute(2, 1, 0)
    kv.read(ko, vo, cache, slots)
    assert np.array_equal(ko.cpu().numpy(), A.values(k, Q8).astype(np.float32))
    assert np.array_equal(vo.cpu().numpy(), A.values(v, Q4).astype(np.float32))
    only = torch.zeros(T, H, D, device=DEV)
    kv.read(None, only, cache, slots)
    assert torch.equal(only, vo)
    buf = torch.cat([torch.zeros(5, device=DEV), _gpu(k).flatten()])
    kv.write(cache, (buf, vx.TensorLayout((T, H, D), (H * D, D, 1), 3, 5)), _gpu(v), slots)
    kv.read(only, None, cache, slots)
    assert torch.equal(only, ko)
    none = torch.empty(0, H, D, device=DEV)
    kv.write(cache, none, none, _i32(np.zeros(0)))
    kv.read(none, none, cache, _i32(np.zeros(0)))


# ------------------------------------------------------------- attention
@pytest.mark.parametrize("types", TYPES, ids=["k8v8", "k8v4", "k4v8", "k4v4"])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("group,page", [(1, 16), (4, 32), (7, 64)])
def test_single_tokens(kv, types, dim, group, page):
    note(f"single {types} {dim} {group} {page}")
    rng = np.random.default_rng(dim + group)
    Batch(kv, rng, [1, 2, 31, 32, 33, 64, 150, 577], [1] * 8, 2, group, dim, page, types).check(kv)


@pytest.mark.parametrize("types", TYPES, ids=["k8v8", "k8v4", "k4v8", "k4v4"])
@pytest.mark.parametrize("dim,heads,group", [(64, 1, 1), (96, 2, 3), (128, 1, 8), (256, 1, 2)])
def test_prompts(kv, types, dim, heads, group):
    note(f"prompts {types} {dim} {heads} {group}")
    rng = np.random.default_rng(dim)
    Batch(kv, rng, [1, 37, 200, 90], [1, 37, 130, 17], heads, group, dim, 32, types).check(kv)


OPTIONS = {
    "all_keys": dict(causal=False),
    "scale": dict(scale=-0.3),
    "cap": dict(softcap=2.0),
    "cap_large": dict(softcap=50.0, scale=1.5),
    "slopes": dict(slopes=True),
    "window": dict(window=19),
    "window_one": dict(window=1),
    "window_both": dict(window=23, causal=False, slopes=True),
    "prefix": dict(prefix=[0, 60, 11]),
    "prefix_window": dict(prefix=[7, 200, 80], window=40),
    "first": dict(first=True),
    "all": dict(first=True, prefix=[5, 70, 90], window=55, softcap=8.0, slopes=True),
}


def _options(rng, o, batch):
    o = dict(o)
    if o.get("slopes"):
        o["slopes"] = rng.uniform(0.01, 0.5, batch.q_heads).astype(np.float32)
    if o.get("first"):  # some see nothing: their document begins behind them
        o["first"] = rng.integers(0, max(batch.lens), batch.T)
    return o


@pytest.mark.parametrize("name", list(OPTIONS))
@pytest.mark.parametrize("dim,types,queries", [(64, (Q8, Q4), [1, 1, 1]), (128, (Q8, Q8), [3, 70, 40]), (96, (Q4, Q4), [64, 130, 33])])
def test_options(kv, name, dim, types, queries):
    note(f"options {name} {dim} {types} {queries}")
    rng = np.random.default_rng(len(name))
    b = Batch(kv, rng, [64, 190, 97], queries, 2, 3, dim, 16, types)
    b.check(kv, **_options(rng, OPTIONS[name], b))


@pytest.mark.parametrize("lens,queries", [([0, 5], [1, 1]), ([0, 0], [3, 2]), ([3, 40], [9, 50]), ([17, 20, 0], [0, 4, 0])],
                         ids=["no_keys", "none_at_all", "more_queries_than_keys", "no_queries"])
def test_rows_that_see_nothing_are_zero(kv, lens, queries):
    rng = np.random.default_rng(1)
    b = Batch(kv, rng, lens, queries, 2, 2, 64, 16, (Q8, Q8))
    b.check(kv)
    b.check(kv, causal=False, first=np.full(b.T, 30))


def test_long_history_is_split_and_joined(kv):
    rng = np.random.default_rng(9)
    b = Batch(kv, rng, [9000, 70, 4097], [1, 1, 1], 1, 4, 128, 64, (Q8, Q4))
    plan = b.check(kv, softcap=20.0)
    assert plan.ws_bytes > 16
    split = b.out.clone()
    plan.ws = None  # without a workspace the keys are not split
    q = _gpu(b.q)
    kv.attend(b.out, (q.flatten(), vx.TensorLayout(tuple(q.shape), tuple(q.stride()), 3)), plan)
    assert (split - b.out).abs().max() < 2e-6
    b.check(kv, window=1000, slopes=rng.uniform(0, 0.01, 4).astype(np.float32))
    b.check(kv, window=3000, causal=False, first=[8100, 0, 5000])


@pytest.mark.parametrize("types", [(Q8, Q8), (Q4, Q4)], ids=["k8v8", "k4v4"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens,queries", [([1], [1]), ([40, 33], [9, 33]), ([300, 70, 129], [40, 5, 64])])
def test_trees(kv, types, dim, lens, queries):
    note(f"trees {types} {dim} {lens} {queries}")
    rng = np.random.default_rng(dim + len(lens))
    b = Batch(kv, rng, lens, queries, 2, 3, dim, 16, types)
    trees = [_tree(rng, n) for n in queries]
    b.check(kv, trees=trees)
    b.check(kv, trees=trees, softcap=5.0, slopes=rng.uniform(0.01, 0.5, b.q_heads).astype(np.float32), window=13)


def test_tree_rows_may_be_empty_or_anything(kv):
    rng = np.random.default_rng(2)
    b = Batch(kv, rng, [30, 45], [30, 40], 1, 2, 64, 16, (Q8, Q8))
    trees = [rng.random((n, n)) < 0.3 for n in b.n]
    trees[0][4] = False  # no key at all
    trees[1][7] = False  # cached keys only
    b.check(kv, trees=trees)
    b.check(kv, trees=trees, first=np.full(b.T, 3), window=30)


def test_tree_mask_from_parents(kv):
    rng = np.random.default_rng(12)
    parents = [[-1, 0, 0, 1, -1, 4], list(range(-1, 39))]
    want = []
    for p in parents:
        t = np.eye(len(p), dtype=bool)
        for j, x in enumerate(p):
            if x >= 0:
                t[j] |= t[x]
        want.append(t)
    assert torch.equal(vx.tree_mask(parents), _words(want))
    b = Batch(kv, rng, [50, 40], [6, 40], 1, 2, 64, 16, (Q8, Q8))
    b.check(kv, trees=want)
    # a chain is a causal chunk (the second sequence)
    plan, out = b.plan(kv), torch.empty(b.q.shape, device=DEV)
    kv.attend(out, _gpu(b.q), plan)
    assert torch.allclose(out[6:], b.out[6:], rtol=0, atol=2e-6)
    with pytest.raises(vx.VortxError, match="parent"):
        vx.tree_mask([[0]])


@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e5])
def test_values_of_any_size(kv, size):
    """V's scale: an f16 down to its subnormals; a whole history of other sizes around."""
    rng = np.random.default_rng(4)
    v = [(_normal(rng, L, 2, 64) * size).astype(np.float32) for L in (70, 300)]
    Batch(kv, rng, [70, 300], [5, 40], 2, 2, 64, 16, (Q8, Q8), v=v).check(kv)
    Batch(kv, rng, [70, 300], [5, 40], 2, 2, 64, 16, (Q4, Q4), v=v).check(kv)


@pytest.mark.parametrize("queries", [1, 80])
def test_values_of_all_sizes_in_one_history(kv, queries):
    """Keys of documents with values 2^24 apart, each seen by its own queries only."""
    rng = np.random.default_rng(8)
    sizes = np.where(np.arange(320) < 256, 1e4, 1e-3)
    v = [(_normal(rng, 320, 1, 64) * sizes[:, None, None]).astype(np.float32)]
    b = Batch(kv, rng, [320], [queries], 1, 2, 64, 16, (Q8, Q8), v=v)
    b.check(kv, first=np.where(np.arange(320 - queries, 320) < 256, 0, 256))


@pytest.mark.parametrize("queries,group", [(2, 2), (40, 4), (90, 4)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("side", ["k", "v", "both"])
@pytest.mark.parametrize("types,huge", [((Q8, Q8), 1e6), ((Q4, Q8), 5e4)], ids=["k8v8", "k4v8"])
def test_huge_keys_out_of_sight_cost_the_others_nothing(kv, queries, group, dim, side, types, huge):
    """Keys before the document and every other draft are 2^15 or 2^20 larger, and no row sees them."""
    rng = np.random.default_rng(14)
    L = 200 + queries
    k, v = [_normal(rng, L, 1, dim)], [_normal(rng, L, 1, dim)]
    first = 111  # the last of its four keys
    trees = np.zeros((queries, queries), bool)
    trees[np.arange(queries), np.arange(queries)] = True
    trees[:, ::2] = False  # no row sees an even draft
    for x, on in ((k, side != "v"), (v, side != "k")):
        if on:
            x[0][:first] *= np.float32(huge)
            x[0][L - queries:][::2] *= np.float32(huge)
    b = Batch(kv, rng, [L], [queries], 1, group, dim, 16, types, k=k, v=v)
    b.check(kv, trees=[trees], first=np.full(queries, first))


@pytest.mark.parametrize("queries", [2, 90])
def test_a_huge_value_of_no_weight(kv, queries):
    """A key that every row sees with a score far below the others', its value 2^28 larger than theirs."""
    rng = np.random.default_rng(15)
    L = 200 + queries
    k, v = [_normal(rng, L, 1, 64) * np.float32(0.1)], [_normal(rng, L, 1, 64) * np.float32(0.01)]
    b = Batch(kv, rng, [L], [queries], 1, 2, 64, 16, (Q8, Q8), k=k, v=v)
    b.q[..., 0] = 40.0
    k[0][50], v[0][50] = 0.0, 1e6
    k[0][50, 0, 0] = -100.0
    c = Batch(kv, rng, [L], [queries], 1, 2, 64, 16, (Q8, Q8), k=k, v=v)
    want, _ = A.attend(b.q, c.kd, c.vd, c.starts, c.lens)
    _, tol = A.attend(b.q, b.kd, [np.clip(x, -1, 1) for x in b.vd], b.starts, b.lens)
    out = torch.empty(b.q.shape, device=DEV)
    kv.attend(out, _gpu(b.q), c.plan(kv))
    assert (np.abs(out.cpu().numpy() - want) <= tol).all()


@pytest.mark.parametrize("size", [1e-35, 1e-4, 1e30])
def test_queries_of_any_size(kv, size):
    rng = np.random.default_rng(4)
    b = Batch(kv, rng, [70, 300], [5, 40], 2, 2, 64, 16, (Q8, Q8))
    b.q[0] = 0.0
    q = (b.q * np.float32(size)).astype(np.float32)
    b.check(kv, q=q, scale=float(np.float32(0.1 / size)) if size < 1e20 else 1e-31)


@pytest.mark.parametrize("queries", [1, 60])
def test_keys_out_of_sight_never_reach_a_result(kv, queries):
    """NaN and infinities in keys and values: rows that see them have them, others not."""
    rng = np.random.default_rng(11)
    L = 200
    k, v = [_normal(rng, L, 1, 128)], [_normal(rng, L, 1, 128)]
    v[0][20, 0, 40] = np.nan
    v[0][L - queries // 2 - 1, 0, 100] = np.inf
    k[0][30, 0, 5] = np.nan
    b = Batch(kv, rng, [L], [queries], 1, 4, 128, 32, (Q8, Q4), k=k, v=v)
    b.check(kv, first=np.where(np.arange(queries) % 3 == 0, 31, 21 if queries == 1 else 40))
    b.check(kv, first=np.full(queries, 10))
    b.check(kv, window=50)
    if queries > 1:
        b.check(kv, trees=[_tree(rng, queries)], first=np.full(queries, 60))


def test_queries_that_are_not_finite_stay_in_their_rows(kv):
    rng = np.random.default_rng(13)
    b = Batch(kv, rng, [90], [40], 1, 2, 64, 16, (Q8, Q8))
    q = b.q.copy()
    q[3, 0, 7], q[5, 1, 0], q[39, 0, 63] = np.nan, np.inf, -np.inf
    want, tol = A.attend(b.q, b.kd, b.vd, b.starts, b.lens)
    out = torch.empty(q.shape, device=DEV)
    kv.attend(out, _gpu(q), b.plan(kv))
    got = out.cpu().numpy()
    hit = np.zeros(q.shape[:2], bool)
    hit[3, 0] = hit[5, 1] = hit[39, 0] = True
    assert np.isnan(got[hit]).all()
    assert (np.abs(got - want)[~hit] <= tol[~hit]).all()


def test_views_of_any_strides_and_layout_pairs(kv):
    rng = np.random.default_rng(14)
    b = Batch(kv, rng, [80, 31], [20, 31], 2, 2, 64, 16, (Q8, Q8))
    plan = b.check(kv)
    want = b.out.clone()
    q = _gpu(b.q)
    T, H, D = q.shape
    q2 = q.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    out = torch.full((H, T, D + 1), float("nan"), device=DEV).permute(1, 0, 2)
    kv.attend(out[..., :D], q2, plan)
    assert torch.equal(out[..., :D], want) and torch.isnan(out[..., D]).all()
    buf = torch.cat([torch.zeros(3, device=DEV), q.flatten()])
    out2 = torch.empty(T * H * D, device=DEV)
    kv.attend((out2, vx.TensorLayout((T, H, D), (H * D, D, 1), 3, 0)), (buf, vx.TensorLayout((T, H, D), (H * D, D, 1), 3, 3)), plan)
    assert torch.equal(out2.view(T, H, D), want)


def test_offsets_beyond_32_bits(kv):
    """Pages past 4 GiB (and past 2^31 values) of a cache."""
    rng = np.random.default_rng(15)
    page, heads, dim = 256, 8, 128
    pages = (5 << 30) // (page * heads * dim // 32 * 68) + 1
    cache = vx.KvCache(pages, page, heads, dim)
    table = np.array([[pages - 1, 1]], np.int32)
    L = 300
    pos = np.arange(L)
    slots = _i32(table[0, pos // page].astype(np.int64) * page + pos % page)
    k, v, q = _normal(rng, L, heads, dim), _normal(rng, L, heads, dim), _normal(rng, 1, heads, dim)
    kv.write(cache, _gpu(k), _gpu(v), slots)
    ko, vo = torch.empty(L, heads, dim, device=DEV), torch.empty(L, heads, dim, device=DEV)
    kv.read(ko, vo, cache, slots)
    kd, vd = A.values(k, Q8), A.values(v, Q8)
    assert np.array_equal(ko.cpu().numpy(), kd.astype(np.float32)) and np.array_equal(vo.cpu().numpy(), vd.astype(np.float32))
    plan = kv.plan(cache, _i32(table), _i32([L]), _i32([0, 1]), q_heads=heads, max_queries=1, max_len=L)
    out = torch.empty(1, heads, dim, device=DEV)
    kv.attend(out, _gpu(q), plan)
    want, tol = A.attend(q, [kd], [vd], [0, 1], [L])
    assert (np.abs(out.cpu().numpy() - want) <= tol).all()


def test_bounds_hold_whatever_the_arrays_say(kv):
    """Lengths, starts and pages out of range are brought into it: nothing is
    read or written outside the operands."""
    rng = np.random.default_rng(16)
    b = Batch(kv, rng, [60], [4], 1, 2, 64, 16, (Q8, Q8))
    out = torch.full((6, 2, 64), 7.0, device=DEV)
    q = _gpu(_normal(rng, 6, 2, 64))
    for table, lens, starts in [([[-5, 2 ** 31 - 1, 3, 0]], [60], [0, 4]), (b.table, [10 ** 9], [0, 4]), (b.table, [-3], [0, 4]),
                                (b.table, [60], [-9, 100]), (b.table, [60], [4, 2])]:
        plan = kv.plan(b.cache, _i32(table), _i32(lens), _i32(starts), q_heads=2, max_queries=4, max_len=60)
        kv.attend(out, q, plan)
    torch.cuda.synchronize()
    assert (out[4:] == 7.0).all()  # queries past max_queries are not computed


def test_same_bits_every_time_and_on_another_stream(kv):
    rng = np.random.default_rng(17)
    b = Batch(kv, rng, [3000, 500], [1, 9], 2, 4, 128, 64, (Q8, Q8))
    plan, q = b.plan(kv), _gpu(b.q)
    outs = [torch.empty(b.q.shape, device=DEV) for _ in range(3)]
    kv.attend(outs[0], q, plan)
    kv.attend(outs[1], q, plan)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    kv.attend(outs[2], q, plan, stream=stream)
    stream.synchronize()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_graph_replays_on_new_lengths(kv):
    """One captured step (write, attend), replayed as the sequences grow."""
    rng = np.random.default_rng(18)
    b = Batch(kv, rng, [700, 40], [1, 1], 2, 2, 64, 16, (Q8, Q8))
    k, v, q, out = (torch.empty(2, h, 64, device=DEV) for h in (2, 2, 4, 4))
    lens, slots = _i32([1, 1]), _i32([-1, -1])
    plan = kv.plan(b.cache, _i32(b.table), lens, _i32(b.starts), q_heads=4, max_queries=1, max_len=700)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        kv.write(b.cache, k, v, slots)
        kv.attend(out, q, plan)
    for step in (0, 17, 699):
        at = [step, min(step, 39)]
        new = [_normal(rng, 2, h, 64) for h in (2, 2, 4)]
        for t, x in zip((k, v, q), new):
            t.copy_(_gpu(x))
        for s in range(2):
            b.kd[s][at[s]], b.vd[s][at[s]] = A.values(new[0][s], Q8), A.values(new[1][s], Q8)
        slots.copy_(_i32([int(b.slots(s, np.array(at[s]))) for s in range(2)]))
        lens.copy_(_i32([a + 1 for a in at]))
        graph.replay()
        torch.cuda.synchronize()
        want, tol = A.attend(new[2], [x[:a + 1] for x, a in zip(b.kd, at)], [x[:a + 1] for x, a in zip(b.vd, at)], b.starts, [a + 1 for a in at])
        assert (np.abs(out.cpu().numpy() - want) <= tol).all(), step


# --------------------------------------------------------------- refusals
def test_refusals(kv):
    f = lambda *s: torch.zeros(*s, device=DEV)  # noqa: E731
    status = lambda e: e.value.status  # noqa: E731
    cache = vx.KvCache(4, 16, 2, 64)
    k, slots = f(3, 2, 64), _i32([0, 1, 2])
    for bad, want in [((f(3, 2, 96), k), _ffi.VX_ERR_SHAPE), ((f(3, 3, 64), f(3, 3, 64)), _ffi.VX_ERR_SHAPE),
                      ((f(4, 2, 64), k), _ffi.VX_ERR_SHAPE), ((f(2, 3, 2, 64), f(2, 3, 2, 64)), _ffi.VX_ERR_SHAPE)]:
        with pytest.raises(vx.VortxError) as e:
            kv.write(cache, *bad, slots)
        assert status(e) == want
    with pytest.raises(vx.VortxError, match="slots"):
        kv.write(cache, k, k, _i32([0, 1]))
    with pytest.raises(TypeError):
        kv.write(cache, k, k, torch.zeros(3, device=DEV, dtype=torch.int64))
    with pytest.raises(TypeError):
        kv.write(cache, k.half(), k, slots)
    with pytest.raises(vx.VortxError, match="zero stride"):
        kv.read(f(1, 2, 64).expand(3, 2, 64), None, cache, slots)
    with pytest.raises(vx.VortxError, match="buffer"):
        vx.KvCache(4, 16, 2, 64, data=torch.zeros(100, dtype=torch.uint8, device=DEV))
    args = (cache, _i32([[0, 1]]), _i32([20]), _i32([0, 3]))
    fine = dict(q_heads=4, max_queries=3, max_len=32)
    for change, want in [(dict(q_heads=3), _ffi.VX_ERR_SHAPE), (dict(softcap=-1.0), _ffi.VX_ERR_INVALID),
                         (dict(softcap=float("nan")), _ffi.VX_ERR_INVALID), (dict(scale=float("inf")), _ffi.VX_ERR_INVALID),
                         (dict(slopes=f(3)), _ffi.VX_ERR_SHAPE), (dict(prefix=_i32([1, 2])), _ffi.VX_ERR_SHAPE),
                         (dict(max_len=2 ** 31), _ffi.VX_ERR_UNSUPPORTED)]:
        with pytest.raises(vx.VortxError) as e:
            kv.plan(*args, **{**fine, **change})
        assert status(e) == want, change
    plan = kv.plan(*args, **fine)
    q = f(3, 4, 64)
    for out, qq, want in [(f(3, 4, 64), f(3, 2, 64), _ffi.VX_ERR_SHAPE), (f(2, 4, 64), q, _ffi.VX_ERR_SHAPE),
                          (f(3, 4, 96), f(3, 4, 96), _ffi.VX_ERR_SHAPE), (f(1, 4, 64).expand(3, 4, 64), q, _ffi.VX_ERR_INVALID)]:
        with pytest.raises(vx.VortxError) as e:
            kv.attend(out, qq, plan)
        assert status(e) == want
    with pytest.raises(vx.VortxError) as e:  # 2 words hold 64 drafts
        kv.attend_tree(f(3, 4, 64), q, kv.plan(*args, q_heads=4, max_queries=70, max_len=32, tokens=3), _i32(np.zeros((3, 2))))
    assert status(e) == _ffi.VX_ERR_SHAPE
    with pytest.raises(vx.VortxError, match="tree"):
        kv.attend_tree(f(3, 4, 64), q, plan, _i32(np.zeros((2, 1))))
    with pytest.raises(vx.VortxError, match="first"):
        kv.attend(f(3, 4, 64), q, kv.plan(*args, **fine, first=_i32([0, 0])))
    for queries, tokens in [(1, 1), (40, 40)]:  # a workspace that is a byte short
        many = kv.plan(vx.KvCache(64, 64, 2, 64), _i32([list(range(64))]), _i32([20]), _i32([0, tokens]), q_heads=4,
                       max_queries=queries, max_len=4096)
        assert many.ws_bytes > 16
        many.ws_bytes -= 1
        q = f(tokens, 4, 64)
        with pytest.raises(vx.VortxError, match="workspace") as e:
            kv.attend((q.flatten(), vx.TensorLayout(tuple(q.shape), tuple(q.stride()), 3)), q, many)
        assert status(e) == _ffi.VX_ERR_INVALID
