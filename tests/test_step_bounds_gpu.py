"""Pages whose counts, lengths and table entries no call left there: nothing but the
arrays' own entries is written. All arrays lie in one buffer, with marks between
them and between the table's rows."""
import ctypes as C

import numpy as np
import pytest
import torch

import vortx_amd as vx
from tests.helpers import note
from vortx_amd import _ffi

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
MARK, GAP = 0x5A5A5A5A, 67


class Arrays:
    """Arrays of the given sizes in one buffer, GAP marks around each; of a table, rows with `apart` entries between their beginnings."""

    def __init__(self, seqs, cols, apart, pages, tokens):
        self.shape = (seqs, cols, apart)
        sizes = {"table": (seqs - 1) * apart + cols if seqs else 0, "lens": seqs, "free": pages, "count": 1, "want": seqs, "starts": seqs + 1,
                 "slots": tokens, "positions": tokens}
        self.at, n = {}, GAP
        for k, size in sizes.items():
            self.at[k] = (n, size)
            n += size + GAP
        self.own = np.zeros(n, bool)
        for k, (a, size) in self.at.items():
            self.own[a:a + size] = True
        a = self.at["table"][0]
        for s in range(seqs):
            self.own[a + s * apart + cols:a + min((s + 1) * apart, self.at["table"][1])] = False
        self.own[self.at["want"][0]:sum(self.at["want"])] = False  # (read only)
        self.host = np.full(n, MARK, np.int32)

    def view(self, k, buf=None):
        a, size = self.at[k]
        return (self.host if buf is None else buf)[a:a + size]

    def table(self, buf=None):
        t, (seqs, cols, apart) = self.view("table", buf), self.shape
        return [t[s * apart:s * apart + cols] for s in range(seqs)]


@pytest.fixture(scope="module")
def kv():
    assert torch.cuda.is_available()
    return vx.KvAttention(0)


def _resize(kv, a, page, pages, tokens):
    buf = torch.tensor(a.host, device=DEV)
    at = {k: buf.data_ptr() + 4 * first for k, (first, _) in a.at.items()}
    seqs, cols, apart = a.shape
    p = _ffi.VxKvPages(at["table"], at["lens"], at["free"], at["count"], seqs, cols, apart, page, pages, 0)
    st = vx.lib().vx_kv_resize(kv._h, torch.cuda.current_stream().cuda_stream, C.byref(p), at["want"], at["starts"], at["slots"], at["positions"], tokens)
    assert st == 0, vx.lib().vx_last_error_message()
    torch.cuda.synchronize()
    got = buf.cpu().numpy()
    assert (got[~a.own] == a.host[~a.own]).all(), np.argwhere(got[~a.own] != a.host[~a.own])[:5]
    return got


ODD = [2 ** 31 - 1, -1, -2 ** 31, 2 ** 30, 0x7FFF0000, 12345, 0, 1]


@pytest.mark.parametrize("seqs,cols,apart,pages,page,tokens", [
    (4, 3, 3, 6, 16, 50), (4, 3, 7, 6, 16, 50), (5, 40, 41, 100, 16, 6000), (300, 9, 13, 1000, 32, 3000), (1100, 6, 9, 5000, 16, 30001),
    (2100, 2, 5, 50, 64, 4096), (1, 1, 1, 1, 16, 1), (3, 2, 4, 0, 16, 20), (0, 3, 5, 4, 16, 9),
])
@pytest.mark.parametrize("count", [2 ** 31 - 1, -7, None])
def test_numbers_that_no_call_left_move_nothing_outside(kv, seqs, cols, apart, pages, page, tokens, count):
    note(f"resize {seqs} x {cols} of {pages} pages, count {count}")
    rng = np.random.default_rng(seqs + cols + pages)
    for turn in range(6):
        a = Arrays(seqs, cols, apart, pages, tokens)
        for row in a.table():
            row[:] = rng.choice(ODD, cols)
        most = cols * page
        a.view("free")[:] = rng.choice(ODD, pages)
        a.view("count")[:] = pages if count is None else count
        a.view("lens")[:] = rng.choice(ODD + [most, most + 1, most - 1], seqs) if turn % 2 else rng.integers(0, most + 1, seqs)
        a.view("want")[:] = rng.choice(ODD + [most, most + 1, 5], seqs) if turn > 1 else rng.integers(-3, most + 3, seqs)
        lens, want = (a.view(k).astype(np.int64) for k in ("lens", "want"))
        got = _resize(kv, a, page, pages, tokens)
        assert 0 <= int(a.view("count", got)[0]) <= pages
        have = np.clip(lens, 0, most)
        after = a.view("lens", got)
        assert ((after == have) | (after == want)).all() and (after <= most).all() and (after >= 0).all()
        new = np.where(want < 0, 0, np.maximum(0, np.where(want < 0, have, want) - have))
        ends = np.minimum(np.concatenate([[0], np.cumsum(new)]), 2 ** 31 - 1)
        assert (a.view("starts", got) == ends).all()
        end = min(int(ends[-1]), tokens)
        assert (a.view("slots", got)[end:] == -1).all() and (a.view("positions", got)[end:] == 0).all()
        # positions of the tokens there are entries for: those of each sequence's in turn
        owner = np.searchsorted(ends[1:], np.arange(end), side="right")
        assert (a.view("positions", got)[:end] == have[owner] + np.arange(end) - ends[owner]).all() if end else True


def test_tables_with_room_between_rows(kv):
    """What a table of wider rows gets is what one without room gets."""
    rng = np.random.default_rng(0)
    seqs, cols, pages, page, tokens = 50, 12, 700, 16, 5000
    wide, tight = Arrays(seqs, cols, 29, pages, tokens), Arrays(seqs, cols, cols, pages, tokens)
    for a in (wide, tight):
        for row in a.table():
            row[:] = 0
        a.view("free")[:] = np.arange(pages)
        a.view("count")[:] = pages
        a.view("lens")[:] = 0
    for _ in range(5):
        want = rng.integers(0, cols * page + 1, seqs)
        outs = []
        for a in (wide, tight):
            a.view("want")[:] = want
            a.host = _resize(kv, a, page, pages, tokens)
            outs.append([np.concatenate(a.table())] + [a.view(k) for k in ("lens", "count", "starts", "slots", "positions")] + [a.view("free")[:int(a.view("count")[0])]])
        assert all((x == y).all() for x, y in zip(*outs))
