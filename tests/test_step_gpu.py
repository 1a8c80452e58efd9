"""Pages of a step, and queries and keys normed and rotated, against plain
restatements: lists of pages, and numpy in 64 bits."""
import numpy as np
import pytest
import torch

import vortx_amd as vx
from tests.helpers import note
from vortx_amd import _ffi

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
Q8, Q4 = vx.VX_Q8_0, vx.VX_Q4_0


@pytest.fixture(scope="module")
def kv():
    assert torch.cuda.is_available()
    return vx.KvAttention(0)


def _i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)


# ----------------------------------------------------------------- pages
class Model:
    """Pages in lists, as vx_kv_resize says it."""

    def __init__(self, pages, page, seqs, cols):
        self.page, self.cols, self.total = page, cols, pages
        self.stack, self.held, self.lens = list(range(pages - 1, -1, -1)), [[] for _ in range(seqs)], [0] * seqs

    def resize(self, want):
        need = lambda n: -(-n // self.page)  # noqa: E731
        before, seqs = list(self.lens), len(self.lens)
        want = [b if w < 0 else w for w, b in zip(want, before)]
        fits = [need(w) <= self.cols for w in want]
        for s in reversed(range(seqs)):
            while len(self.held[s]) > need(want[s]):
                self.stack.append(self.held[s].pop())
        room, asked, starts, slots, pos = len(self.stack), 0, [0], [], []
        for s in range(seqs):
            more = max(0, need(want[s]) - len(self.held[s])) if fits[s] else 0
            asked += more
            served = fits[s] and (more == 0 or asked <= room)
            if served:
                for _ in range(more):
                    self.held[s].append(self.stack.pop())
                self.lens[s] = want[s]
            new = range(before[s], want[s])
            pos += new
            slots += [self.held[s][p // self.page] * self.page + p % self.page if served else -1 for p in new]
            starts.append(len(pos))
        return starts, slots, pos


def _check(pages, step, model, want, said):
    starts, slots, pos = said
    cap = step.tokens
    pad = lambda a, v: (a + [v] * cap)[:cap]  # noqa: E731
    assert step.starts.tolist() == starts
    assert step.slots.tolist() == pad(slots, -1)
    assert step.positions.tolist() == pad(pos, 0)
    assert pages.lens.tolist() == model.lens
    n = int(pages.free_count)
    assert pages.free[:n].tolist() == model.stack
    table = pages.table.tolist()
    for row, held in zip(table, model.held):
        assert row[:len(held)] == held
    assert sorted(model.stack + sum(model.held, [])) == list(range(model.total))


@pytest.mark.parametrize("seqs,cols,page,pages,most,cap", [
    (1, 4, 16, 4, 64, 64),           # one sequence, to the last slot
    (1, 1, 16, 1, 16, 1),            # a single page, more tokens than the step has entries
    (3, 40, 16, 60, 400, 700),       # too few pages now and then
    (32, 9, 256, 500, 2300, 5000),   # slots in a launch of their own
    (65, 300, 16, 9000, 4800, 30000),
    (1024, 5, 16, 2500, 60, 4096),
    (1025, 5, 16, 5125, 80, 4097),   # a second round of 1024
    (2600, 3, 32, 4000, 90, 4000),   # a third, and too few pages
])
def test_pages_grow_and_shrink(kv, seqs, cols, page, pages, most, cap):
    rng = np.random.default_rng(seqs * 1000 + cols)
    p, step, model = vx.KvPages(pages, page, seqs, cols), vx.KvStep(seqs, cap), Model(pages, page, seqs, cols)
    for turn in range(7):
        note(f"resize {seqs} sequences, turn {turn}")
        want = rng.integers(0, most + 1, seqs)
        kind = rng.integers(0, 6, seqs)
        lens = np.array(model.lens)
        want = np.where(kind == 0, 0, np.where(kind == 1, -rng.integers(1, 9, seqs), np.where(kind == 2, lens, np.where(kind == 3, lens + 1, want))))
        if turn == 3:
            want[rng.integers(0, seqs)] = cols * page + 1  # a row too short
        if turn == 4:
            want[:] = 0
        kv.resize(p, _i32(want), step)
        _check(p, step, model, want, model.resize([int(w) for w in want]))


def test_a_step_taken_back_leaves_everything_as_it_was(kv):
    rng = np.random.default_rng(5)
    p, step = vx.KvPages(400, 16, 40, 30), vx.KvStep(40, 6000)
    have = _i32(rng.integers(0, 160, 40))
    kv.resize(p, have, step)
    lens, free, count, table = (t.clone() for t in (p.lens, p.free, p.free_count, p.table))
    assert torch.equal(lens, have)
    for turn in range(4):
        kv.resize(p, _i32(rng.integers(0, 200, 40)), step)
        kv.resize(p, lens, step)
        n = int(count)
        assert torch.equal(p.lens, lens) and torch.equal(p.free_count, count) and torch.equal(p.free[:n], free[:n])
        for s, L in enumerate(lens.tolist()):
            assert torch.equal(p.table[s, :-(-L // 16)], table[s, :-(-L // 16)])


@pytest.mark.parametrize("want", [2 ** 31 - 1, 2 ** 31 - 17, 1 << 30])
def test_lengths_past_everything(kv, want):
    p, step = vx.KvPages(10, 65536, 3, 2), vx.KvStep(3, 5)
    kv.resize(p, _i32([want, 7, want]), step)
    assert p.lens.tolist() == [0, 7, 0] and int(p.free_count) == 9 and p.table[1, 0] == 0
    # the first one's tokens take all entries of the step
    assert step.slots.tolist() == [-1] * 5 and step.positions.tolist() == [0, 1, 2, 3, 4]
    assert step.starts.tolist() == [0, want, min(want + 7, 2 ** 31 - 1), min(2 * want + 7, 2 ** 31 - 1)]


def test_pages_without_sequences_or_pages(kv):
    p, step = vx.KvPages(4, 16, 0, 0), vx.KvStep(0, 3)
    kv.resize(p, _i32([]), step)
    assert step.starts.tolist() == [0] and step.slots.tolist() == [-1] * 3 and int(p.free_count) == 4
    p, step = vx.KvPages(0, 16, 2, 3), vx.KvStep(2, 0)
    kv.resize(p, _i32([5, 0]), step)
    assert step.starts.tolist() == [0, 5, 5] and p.lens.tolist() == [0, 0] and int(p.free_count) == 0


def test_counts_that_no_call_left_are_bounded(kv):
    """A free count or lengths out of range: nothing outside the arrays is touched."""
    p, step = vx.KvPages(6, 16, 4, 3), vx.KvStep(4, 50)
    guard = torch.full((64,), 77, dtype=torch.int32, device=DEV)
    p.free_count.fill_(2 ** 31 - 1)
    p.lens.copy_(_i32([2 ** 31 - 1, -5, 40, 1000]))
    kv.resize(p, _i32([0, 20, 0, -1]), step)
    assert 0 <= int(p.free_count) <= 6 and p.lens.tolist()[:3] == [0, 20, 0] and p.lens.tolist()[3] <= 48
    assert (guard == 77).all()


def test_pages_in_a_captured_graph(kv):
    rng = np.random.default_rng(8)
    p, step, model = vx.KvPages(300, 16, 20, 20), vx.KvStep(20, 5000), Model(300, 16, 20, 20)
    want = _i32(np.zeros(20))
    kv.resize(p, want, step)  # (loads the code before the capture)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        kv.resize(p, want, step)
    for _ in range(5):
        w = rng.integers(0, 260, 20)
        want.copy_(_i32(w))
        graph.replay()
        torch.cuda.synchronize()
        _check(p, step, model, w, model.resize([int(x) for x in w]))


def test_pages_refusals(kv):
    p, step = vx.KvPages(4, 16, 2, 2), vx.KvStep(2, 3)
    for bad, error in [(torch.zeros(2), TypeError), (_i32([1, 2, 3]), vx.VortxError), (_i32([[1], [2]])[:, 0:1], vx.VortxError),
                       (_i32([1, 9, 2, 9])[::2], vx.VortxError), (torch.zeros(2, dtype=torch.int32), TypeError)]:
        with pytest.raises(error):
            kv.resize(p, bad, step)
    with pytest.raises(vx.VortxError):
        kv.resize(p, _i32([1, 1]), vx.KvStep(3, 3))
    with pytest.raises(vx.VortxError):
        vx.KvPages(4, 16, -1, 2)
    bad = vx.KvPages(4, 24, 2, 2)
    with pytest.raises(vx.VortxError):
        kv.resize(bad, _i32([1, 1]), step)


# ----------------------------------------------------------------- rotation
def _rotated(x, pos, freqs, pairs, norm, w, eps):
    """[T, H, D] in 64 bits."""
    y = x.astype(np.float64)
    if norm:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + np.float64(np.float32(eps)))
        if w is not None:
            y = y * w.astype(np.float64)
    r = 0 if freqs is None else 2 * len(freqs)
    out = y.copy()
    if r:
        t = (pos.astype(np.float64)[:, None] * freqs)[:, None, :]
        a, b = (slice(0, r, 2), slice(1, r, 2)) if pairs else (slice(0, r // 2), slice(r // 2, r))
        out[..., a] = y[..., a] * np.cos(t) - y[..., b] * np.sin(t)
        out[..., b] = y[..., b] * np.cos(t) + y[..., a] * np.sin(t)
    return out


def _close(got, ref):
    """One rounding to f32 of a result in f64: half a step, 2^-24 of the value
    (2^-149 below the normal numbers), and what some twenty f64 roundings of numbers up to the row's
    largest leave: 2^-48 of that."""
    got = got.cpu().numpy().astype(np.float64)
    top = np.abs(ref).max(-1, keepdims=True)
    off = np.abs(got - ref) - (np.abs(ref) * 2.0 ** -24 + 2.0 ** -149 + top * 2.0 ** -48)
    assert np.isfinite(got).all() and (off <= 0).all(), float(off.max())


POSITIONS = [0, 1, 2, 7, 1000, 131071, 1000003, 2 ** 31 - 1, -1, -77]


@pytest.mark.parametrize("dim,rotated,pairs,norm,weight", [
    (64, 64, False, True, "shared"), (128, 128, False, True, "heads"), (256, 256, False, True, "shared"), (96, 96, False, False, None),
    (128, 128, True, True, "shared"), (80, 48, True, False, None), (80, 48, False, True, "heads"), (112, 112, False, True, None),
    (2, 2, False, True, "shared"), (2, 2, True, False, None), (1, 0, False, True, "heads"), (6, 4, False, True, "shared"),
    (30, 30, True, True, "heads"), (30, 22, False, True, "shared"), (250, 130, False, True, "heads"), (255, 254, True, True, "shared"),
    (192, 0, False, True, "heads"), (64, 12, False, False, None), (68, 64, False, True, "shared"), (24, 24, True, True, "shared"),
])
@pytest.mark.parametrize("tokens,hq,hk", [(1, 1, 1), (10, 4, 2), (333, 5, 3)])
def test_rotate(kv, dim, rotated, pairs, norm, weight, tokens, hq, hk):
    note(f"rotate {tokens} x {hq} + {hk} x {dim}, {rotated} rotated, pairs {pairs}, norm {norm}, weight {weight}")
    rng = np.random.default_rng(dim * 7 + rotated + tokens)
    q, k = (rng.standard_normal((tokens, h, dim)).astype(np.float32) for h in (hq, hk))
    pos = np.array((POSITIONS * (tokens // 10 + 1))[:tokens], np.int64)
    freqs = 10000.0 ** (-np.arange(rotated // 2) * 2 / max(rotated, 1)) if rotated else None
    ws = [None, None]
    if weight:
        ws = [(1 + 0.3 * rng.standard_normal((h, dim) if weight == "heads" else (dim,))).astype(np.float32) for h in (hq, hk)]
    up = lambda a: None if a is None else torch.tensor(a, device=DEV)  # noqa: E731
    how = kv.rotation(up(freqs), pairs=pairs, norm=norm, q_weight=up(ws[0]), k_weight=up(ws[1]), eps=1e-6)
    refs = [_rotated(x, pos, freqs, pairs, norm, w, 1e-6) for x, w in ((q, ws[0]), (k, ws[1]))]
    gq, gk = up(q), up(k)
    qo, ko = torch.full_like(gq, float("nan")), torch.full_like(gk, float("nan"))
    kv.rotate(qo, gq, ko, gk, _i32(pos), how)
    _close(qo, refs[0])
    _close(ko, refs[1])
    # views of one projection's rows (odd offsets and strides too), heads before tokens, in place: the same bits
    both = torch.empty(tokens, (hq + hk) * dim + 3, device=DEV)
    vq, vk = both[:, 1:1 + hq * dim].unflatten(1, (hq, dim)), both[:, 1 + hq * dim:1 + (hq + hk) * dim].unflatten(1, (hk, dim))
    vq.copy_(gq), vk.copy_(gk)
    both[:, 0] = both[:, -2:].fill_(5.0)[:, 0]
    kv.rotate(vq, vq, vk, vk, _i32(pos), how)
    assert torch.equal(vq, qo) and torch.equal(vk, ko) and (both[:, 0] == 5).all() and (both[:, -2:] == 5).all()
    tq, tk = gq.transpose(0, 1).contiguous().transpose(0, 1), gk.permute(2, 1, 0).contiguous().permute(2, 1, 0)
    oq = torch.empty(hq, dim, tokens, device=DEV).permute(2, 0, 1)
    ok = torch.empty(hk, tokens, dim, device=DEV).transpose(0, 1)
    kv.rotate(oq, tq, ok, tk, _i32(pos), how)
    assert torch.equal(oq, qo) and torch.equal(ok, ko)
    # queries alone
    qo2 = torch.empty_like(qo)
    kv.rotate(qo2, gq, None, None, _i32(pos), how)
    assert torch.equal(qo2, qo)


def test_norm_of_very_large_and_small_rows(kv):
    rng = np.random.default_rng(3)
    scale = np.array([1e-38, 1e-30, 1e-10, 1.0, 1e10, 1e30, 1e38], np.float32)
    q = (rng.uniform(-1, 1, (7, 2, 128)).astype(np.float32) * scale[:, None, None]).astype(np.float32)
    how = kv.rotation(vx.rotation_freqs(128), norm=True, eps=0.0)
    pos = np.arange(7)
    qo = torch.empty(7, 2, 128, device=DEV)
    kv.rotate(qo, torch.tensor(q, device=DEV), None, None, _i32(pos), how)
    _close(qo, _rotated(q, pos, 10000.0 ** (-np.arange(64) / 64), False, True, None, 0.0))


def test_rows_that_are_not_finite_stay_by_themselves(kv):
    rng = np.random.default_rng(4)
    q = torch.tensor(rng.standard_normal((3, 4, 64)).astype(np.float32), device=DEV)
    how = kv.rotation(vx.rotation_freqs(32), norm=True)
    good, bad = torch.empty_like(q), torch.empty_like(q)
    kv.rotate(good, q, None, None, _i32([3, 4, 5]), how)
    q[1, 2, 7], q[2, 0, 50], q[0, 0] = float("nan"), float("inf"), 0.0
    kv.rotate(bad, q, None, None, _i32([3, 4, 5]), how)
    assert bad[1, 2].isnan().all() and (bad[0, 0] == 0).all() and bad[2, 0, 50].isnan() and (bad[2, 0, :50] == 0).all()
    for t, h in ((0, 1), (0, 2), (1, 0), (1, 1), (1, 3), (2, 1), (2, 3)):
        assert torch.equal(good[t, h], bad[t, h])
    plain = kv.rotation(vx.rotation_freqs(32))  # without a norm the dims that are not rotated are copies
    q[1, 2, 60] = float("-inf")
    kv.rotate(bad, q, None, None, _i32([3, 4, 5]), plain)
    assert torch.equal(bad[:, :, 32:], q[:, :, 32:])


@pytest.mark.parametrize("types", [(Q8, Q8), (Q8, Q4), (Q4, Q8), (Q4, Q4)])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("tokens,order", [(1, "any"), (37, "any"), (301, "runs"), (513, "any"), (259, "runs")])
def test_rows_rotated_into_the_cache(kv, types, dim, tokens, order):
    """The bits of vx_rotate and vx_kv_write one after the other, in every byte of the cache."""
    note(f"write_rotated {tokens} x {dim}, types {types}, {order}")
    rng = np.random.default_rng(tokens + dim)
    hq, hk, page = 6, 3, 32
    pages = tokens // page + 4
    q, k, v = (torch.tensor(rng.standard_normal((tokens, h, dim)).astype(np.float32), device=DEV) for h in (hq, hk, hk))
    w = torch.tensor((1 + 0.2 * rng.standard_normal((hk, dim))).astype(np.float32), device=DEV)
    slots = rng.permutation(pages * page)[:tokens] if order == "any" else 3 + np.arange(tokens)
    if tokens > 30:
        slots[[5, 11, 29]] = [-1, pages * page, 2 ** 31 - 1]
    pos, slots = _i32(rng.integers(0, 100000, tokens)), _i32(slots)
    for pairs, rotated in ((False, dim), (True, dim), (False, dim // 2 + 6)):
        how = kv.rotation(vx.rotation_freqs(rotated), pairs=pairs, norm=True, q_weight=w[0].contiguous(), k_weight=w)
        a, b = vx.KvCache(pages, page, hk, dim, *types), vx.KvCache(pages, page, hk, dim, *types)
        a.data.fill_(171), b.data.fill_(171)
        qo, ko, qf = torch.empty_like(q), torch.empty_like(k), torch.empty_like(q)
        kv.rotate(qo, q, ko, k, pos, how)
        kv.write(a, ko, v, slots)
        kept = k.clone()
        kv.write_rotated(b, qf, q, k, v, pos, slots, how)
        assert torch.equal(qf, qo) and torch.equal(k, kept) and torch.equal(a.data, b.data)
        b.data.fill_(171)
        kv.write_rotated(b, None, None, k, v, pos, slots, how)
        assert torch.equal(a.data, b.data)
        vq = torch.empty(hq, tokens, dim, device=DEV).transpose(0, 1)
        b.data.fill_(171)
        kv.write_rotated(b, vq, q, k.permute(2, 0, 1).contiguous().permute(1, 2, 0), v.transpose(0, 1).contiguous().transpose(0, 1), pos,
                         slots, how)
        assert torch.equal(vq, qo) and torch.equal(a.data, b.data)


def test_rotation_refusals(kv):
    f = vx.rotation_freqs(64)
    w = torch.ones(64, device=DEV)
    q, k = torch.zeros(3, 4, 64, device=DEV), torch.zeros(3, 2, 64, device=DEV)
    pos = _i32([0, 1, 2])
    for make, error in [(lambda: kv.rotation(f.float()), TypeError), (lambda: kv.rotation(f.cpu()), TypeError),
                        (lambda: kv.rotation(f.reshape(2, 16)), vx.VortxError), (lambda: kv.rotation(f[::2]), vx.VortxError),
                        (lambda: kv.rotation(f, norm=True, q_weight=w.double()), TypeError),
                        (lambda: kv.rotation(f, norm=True, q_weight=w, k_weight=w[:32].contiguous()), vx.VortxError)]:
        with pytest.raises(error):
            make()
    norm = kv.rotation(f, norm=True, q_weight=torch.ones(4, 64, device=DEV), k_weight=w)
    for call in [lambda: kv.rotate(q, q, k, k, _i32([0, 1]), norm),                              # too few positions
                 lambda: kv.rotate(q, q, k, k, None, norm),
                 lambda: kv.rotate(q, q, None, k, pos, norm),
                 lambda: kv.rotate(q, q[:2], k, k, pos, norm),
                 lambda: kv.rotate(q[:, :3], q[:, :3], k, k, pos, norm),                         # weights for other heads
                 lambda: kv.rotate(q[..., :32], q[..., :32], k[..., :32], k[..., :32], pos, norm),  # for other dims
                 lambda: kv.rotate(q[0], q[0], None, None, pos, norm),
                 lambda: kv.rotate(q, q, k, k, pos, kv.rotation(vx.rotation_freqs(66))),         # more than a head has
                 lambda: kv.rotate(q, q, k, k, pos, kv.rotation(f, q_weight=w)),                 # a weight without a norm
                 lambda: kv.rotate(q, q, k, k, pos, kv.rotation(f, norm=True, eps=-1.0))]:
        with pytest.raises(vx.VortxError):
            call()
    with pytest.raises(TypeError):
        kv.rotate(q, q, k, k, pos.long(), norm)
    cache = vx.KvCache(2, 16, 2, 64)
    for call in [lambda: kv.write_rotated(cache, q, q, k, k, pos, _i32([0, 1]), norm),
                 lambda: kv.write_rotated(cache, None, q, k, k, pos, pos, norm),
                 lambda: kv.write_rotated(cache, q, q, k, k[:, :1], pos, pos, norm),
                 lambda: kv.write_rotated(cache, q[:2], q[:2], k, k, pos, pos, norm)]:
        with pytest.raises(vx.VortxError):
            call()
    assert _ffi.VX_ROTATE_PAIRS == 1 and _ffi.VX_ROTATE_NORM == 2


@pytest.mark.parametrize("types", [(Q8, Q8), (Q8, Q4)])
def test_slots_past_32_bits_of_bytes(kv, types):
    note(f"far slots {types}")
    hk, dim, page, pages, n = 8, 256, 64, 1 << 15, 45
    g = torch.Generator(device=DEV).manual_seed(3)
    k, v = (torch.randn(n, hk, dim, generator=g, device=DEV) for _ in range(2))
    slots, pos = _i32(pages * page - 3 * np.arange(n) - 1), _i32(np.arange(n) * 999)
    cache, how = vx.KvCache(pages, page, hk, dim, *types), kv.rotation(vx.rotation_freqs(dim), norm=True)
    assert cache.data.numel() > 2 ** 32
    got, want = ([torch.empty_like(k) for _ in range(2)] for _ in range(2))
    turned = torch.empty_like(k)
    kv.rotate(turned, k, None, None, pos, how)
    kv.write(cache, turned, v, slots)
    kv.read(*want, cache, slots)
    kv.write(cache, v, k, slots)
    kv.write_rotated(cache, None, None, k, v, pos, slots, how)
    kv.read(*got, cache, slots)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    many = slots.repeat_interleave(32)[:1400] - (torch.arange(1400, device=DEV) * 97 % 1000 * 512).int()  # (enough to go by fours)
    many = torch.unique(many).flip(0).contiguous()
    k, v = (torch.randn(len(many), hk, dim, generator=g, device=DEV) for _ in range(2))
    pos, turned = _i32(np.arange(len(many))), torch.empty_like(k)
    kv.rotate(turned, k, None, None, pos, how)
    got, want = ([torch.empty_like(k) for _ in range(2)] for _ in range(2))
    kv.write(cache, turned, v, many)
    kv.read(*want, cache, many)
    kv.write(cache, v, k, many)
    kv.write_rotated(cache, None, None, k, v, pos, many, how)
    kv.read(*got, cache, many)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_more_tokens_than_a_launch_takes(kv):
    """2^20 of them a launch: the same as two calls."""
    note("2^20 + 37 tokens")
    n, cut, dim, page = (1 << 20) + 37, 500001, 64, 64
    g = torch.Generator(device=DEV).manual_seed(5)
    q, k, v = (torch.randn(n, 1, dim, generator=g, device=DEV) for _ in range(3))
    pos, slots = torch.arange(n, dtype=torch.int32, device=DEV), torch.arange(n, dtype=torch.int32, device=DEV).flip(0).contiguous()
    how = kv.rotation(vx.rotation_freqs(dim), norm=True)
    a, b = (vx.KvCache(-(-n // page), page, 1, dim) for _ in range(2))
    a.data.fill_(1), b.data.fill_(1)
    qa, ka, qb, kb = (torch.empty_like(q) for _ in range(4))
    kv.rotate(qa, q, ka, k, pos, how)
    for s in (slice(0, cut), slice(cut, n)):
        kv.rotate(qb[s], q[s], kb[s], k[s], pos[s], how)
    assert torch.equal(qa, qb) and torch.equal(ka, kb)
    qa.zero_()
    kv.write_rotated(a, qa, q, k, v, pos, slots, how)
    for s in (slice(0, cut), slice(cut, n)):
        kv.write(b, kb[s], v[s], slots[s])
    assert torch.equal(qa, qb) and torch.equal(a.data, b.data)


def test_other_streams(kv):
    """Rows rotated into two caches at once, each on a stream of its own."""
    note("two streams")
    g = torch.Generator(device=DEV).manual_seed(6)
    n, hq, hk, dim = 600, 8, 2, 128
    q, k, v = (torch.randn(n, h, dim, generator=g, device=DEV) for h in (hq, hk, hk))
    pos, slots = _i32(np.arange(n) + 5), _i32(np.random.default_rng(1).permutation(n))
    how = kv.rotation(vx.rotation_freqs(dim), norm=True, q_weight=torch.rand(dim, generator=g, device=DEV))
    caches, outs = [vx.KvCache(10, 64, hk, dim) for _ in range(3)], [torch.zeros_like(q) for _ in range(3)]
    for c in caches:
        c.data.fill_(9)
    kv.write_rotated(caches[2], outs[2], q, k, v, pos, slots, how)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for s, c, o in zip(streams, caches, outs):
            with torch.cuda.stream(s):
                kv.write_rotated(c, o, q, k, v, pos, slots, how)
    kv.write_rotated(caches[0], outs[0], q, k, v, pos, slots, how, stream=streams[0])
    torch.cuda.synchronize()
    for c, o in zip(caches[:2], outs):
        assert torch.equal(c.data, caches[2].data) and torch.equal(o, outs[2])


def test_calls_through_ctypes_are_the_same(kv, monkeypatch):
    """What the fast calls do not take goes through ctypes: the same results and refusals."""
    note("ctypes")
    g = torch.Generator(device=DEV).manual_seed(9)
    n, hq, hk, dim = 20, 4, 2, 64
    q, k, v = (torch.randn(n, h, dim, generator=g, device=DEV) for h in (hq, hk, hk))
    how = kv.rotation(vx.rotation_freqs(dim), norm=True, q_weight=torch.rand(hq, dim, generator=g, device=DEV))
    i8, w, x = vx.Int8Gemm(0), torch.randn(30, 100, generator=g, device=DEV), torch.randn(9, 100, generator=g, device=DEV)

    def everything():
        pages, step = vx.KvPages(8, 16, 2, 4), vx.KvStep(2, n)
        kv.resize(pages, _i32([13, 6]), step)
        cache = vx.KvCache(8, 16, hk, dim)
        cache.data.zero_()
        qo, ko, qw, out, gated = torch.empty_like(q), torch.empty_like(k), torch.empty_like(q), torch.empty(9, 30, device=DEV), torch.empty(9, 30, device=DEV)
        kv.rotate(qo, q, ko, k, step.positions, how)
        kv.write_rotated(cache, qw, q, k, v, step.positions, step.slots, how)
        rows, xq = vx.Int8Rows.empty(30, 100), vx.Int8Rows.empty(9, 100)
        rows.data.zero_(), xq.data.zero_()
        i8.quantize(rows, w), i8.quantize(xq, x)
        i8.dispatch(out, x, rows, workspace=i8.workspace(9, 100))
        i8.dispatch_gated(gated, xq, rows, rows, "relu")
        for call in [lambda: kv.resize(pages, _i32([1]), step), lambda: kv.rotate(qo, q, ko, k[:3], step.positions, how),
                     lambda: kv.write_rotated(cache, None, None, k, v, step.positions[:3], step.slots, how), lambda: i8.dispatch(out, x, rows),
                     lambda: i8.quantize(rows, x)]:
            with pytest.raises(vx.VortxError):
                call()
        return [pages.table, pages.lens, pages.free_count, step.starts, step.slots, step.positions, cache.data, qo, ko, qw, rows.data, rows.scales,
                xq.data, out, gated]

    fast = everything()
    for name in ("rotate", "kv_write_rotated", "kv_resize", "i8_quantize", "gemm_i8"):
        monkeypatch.setattr(vx._pycall, name, lambda *a: None)
    for a, b in zip(fast, everything()):
        assert torch.equal(a, b)
