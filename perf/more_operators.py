"""What a decoder layer has around its attention, as measurable cases.

`listed()` names twelve cases and `draw()` gives more of the same ranges;
`prepare(case, seed)` makes what a program holds before a call, `run(state)` is
one pass, `exact(case, seed)` the same results in 64 bits and `work(case)` what
a pass cannot do without. With `own` false `run` is the plain form, elementary
torch operations; with `own` true it makes the calls of `vortx_amd`.

Operators (T tokens in S sequences):

* pages: the page table, lengths, starts, slots and positions of a step from
  how many tokens each sequence is to hold; pages come from a stack of free
  ones and go back to it. A pass takes the step and then takes it back (a
  rejected draft, a cancelled batch), so that the next one finds the same;
* rotate: q and k of T tokens, each head normed (x / sqrt(mean x^2 + eps) w)
  and its pairs of dims rotated by position times frequency;
* store: the same, k and v then quantized into slots of the paged cache, and
  what these hold read back;
* product: x [T, K] rounded to 8 bits with a scale for each token, times
  weights [N, K] in 8 bits with a scale for each channel;
* gated: act(x gate^T) (x up^T) of two such products.

8-bit rows: m = max|x|, d = f32(m / 127), q = clamp(rint(x f32(127 / m)),
-127, 127), each operation one f32 rounding; it stands for d q. Blocks of 32 in
the cache: 8 bits, d = f16(max|x| / 127) and q = clamp(rint(x (1 / d)), -127,
127); 4 bits, m the value of the largest magnitude, d = f16(m / -8) and q =
clamp(rint(x (1 / d)), -8, 7).
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False
DEV = "cuda:0"
EPS = 1e-6


# ----------------------------------------------------------------- cases
def _pages(name, seqs, most, grow, page, finish=0.0, spare=1.0):
    return {"name": name, "op": "pages", "seqs": seqs, "most": most, "grow": grow, "page": page, "finish": finish, "spare": spare}


def _rotate(name, tokens, heads, kv_heads, dim, rotated, style, norm, far):
    return {"name": name, "op": "rotate", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotated": rotated,
            "style": style, "norm": norm, "far": far}


def _store(name, tokens, heads, kv_heads, dim, style, norm, far, page, k, v):
    return {"name": name, "op": "store", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotated": dim,
            "style": style, "norm": norm, "far": far, "page": page, "k": k, "v": v}


def _product(name, tokens, rows, cols, op="product", act="", wide=0):
    return {"name": name, "op": op, "tokens": tokens, "rows": rows, "cols": cols, "act": act, "wide": wide}


def listed():
    return [
        # A decode step of a serving batch: a token more for each sequence, now and then a page. Latency.
        _pages("pages_step", 32, 8000, 1, 16),
        # A step with prompts of up to 4000 tokens among 200 sequences, of which some have ended.
        _pages("pages_prompts", 200, 6000, 4000, 64, finish=0.2),
        # One token's queries and keys, normed and rotated. Latency.
        _rotate("rotate_token", 1, 32, 8, 128, 128, "halves", "shared", 9000),
        # A prompt, partly rotated in neighbouring pairs, at far positions.
        _rotate("rotate_prompt", 4097, 16, 16, 80, 48, "pairs", "none", 1000000),
        # A decode step's keys and values into the cache, the queries and keys normed and rotated on the way.
        _store("store_step", 32, 32, 8, 128, "halves", "shared", 9000, 16, "q8_0", "q8_0"),
        # The same for prompts, a norm weight for each head, values in 4 bits.
        _store("store_prompts", 8000, 32, 8, 128, "halves", "heads", 40000, 64, "q8_0", "q4_0"),
        # The smallest product: one token through a projection.
        _product("product_token", 1, 11008, 4096),
        # A decode batch and a short prompt together, through a down projection.
        _product("product_batch", 100, 4096, 11008),
        # A prompt through a projection: the largest call.
        _product("product_prompt", 4096, 11008, 4096),
        # One token through both projections of a gated feed-forward block.
        _product("gated_token", 1, 11008, 4096, "gated", "silu"),
        # A decode batch through them, sizes that are multiples of nothing, x a part of wider rows.
        _product("gated_batch", 13, 5001, 4087, "gated", "gelu_tanh", wide=9),
        # A prompt through them.
        _product("gated_prompt", 2011, 11008, 4096, "gated", "silu"),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["pages", "rotate", "store", "product", "product", "product", "gated", "gated"])
    if op == "pages":
        c = _pages("", _log(rng, 1, 1500), _log(rng, 1, 16000), rng.choice([1, 1, 7, _log(rng, 1, 4000)]), rng.choice([16, 32, 64, 128, 256]),
                   finish=rng.choice([0.0, 0.1, 0.5]), spare=rng.choice([1.0, 1.0, 0.5]))
        while c["seqs"] * c["grow"] > 4e5:
            c["seqs"] = c["seqs"] // 2 + 1
    elif op in ("rotate", "store"):
        kv, group = rng.choice([1, 2, 3, 4, 8, 8, 12]), rng.choice([1, 2, 3, 4, 4, 5, 8])
        dim = rng.choice([64, 96, 128, 128, 256] if op == "store" else [24, 64, 80, 96, 112, 128, 128, 192, 256])
        tokens = _log(rng, 1, 8000)
        while tokens * kv * (group + 2) * dim > 4.9e7:
            tokens = tokens // 2 + 1
        rest = dict(style=rng.choice(["halves", "pairs"]), norm=rng.choice(["none", "shared", "shared", "heads"]), far=_log(rng, 100, 2000000))
        if op == "rotate":
            c = _rotate("", tokens, kv * group, kv, dim, rng.choice([dim, dim, dim // 2, 2 * rng.randint(1, dim // 2)]), **rest)
        else:
            c = _store("", tokens, kv * group, kv, dim, page=rng.choice([16, 32, 64, 128, 256]), k=rng.choice(["q8_0", "q4_0"]),
                       v=rng.choice(["q8_0", "q4_0"]), **rest)
    else:
        most = 1.8e11 / (2 if op == "gated" else 1)
        tokens, rows, cols = _log(rng, 1, 4096), _log(rng, 17, 14336), _log(rng, 64, 14336)
        while tokens * rows * cols > most:
            tokens, rows, cols = tokens * 3 // 4 + 1, rows * 7 // 8 + 1, cols * 7 // 8 + 1
        if rng.random() < 0.5:  # (as models have them)
            rows, cols = -(-rows // 64) * 64, cols // 64 * 64
        c = _product("", tokens, rows, cols, op, rng.choice(["silu", "gelu_tanh", "gelu", "relu"]) if op == "gated" else "",
                     wide=rng.choice([0, 0, 4, 9]))
    del c["name"]
    return c


# ------------------------------------------------ sizes that follow from a case
def _rng(c):
    return random.Random(repr(sorted((k, v) for k, v in c.items() if k != "name")))


class _Held:
    """pages: what the sequences hold before a step, what they are to hold (of the case alone), and which pages are whose."""

    def __init__(self, c, seed):
        rng = _rng(c)
        S, page = c["seqs"], c["page"]
        self.have = [rng.randint(0, c["most"]) for _ in range(S)]
        self.have[0] = c["most"]
        self.want = [h + (1 if c["grow"] == 1 else rng.randint(1, c["grow"])) for h in self.have]
        for s in range(1, S):
            if rng.random() < c["finish"]:
                self.want[s] = 0 if rng.random() < 0.5 else rng.randint(0, self.have[s])
        need = lambda n: -(-n // page)  # noqa: E731
        self.cols = max(need(max(a, b)) for a, b in zip(self.have, self.want)) + 1
        self.old = [need(h) for h in self.have]
        self.new = [need(w) for w in self.want]
        taken = sum(max(0, b - a) for a, b in zip(self.old, self.new))
        given = sum(max(0, a - b) for a, b in zip(self.old, self.new))
        free = 5 + taken if c["spare"] >= 1 else max(0, int(taken * c["spare"]) - given)  # spare < 1: some sequences find none
        self.total = sum(self.old) + free
        order = list(range(self.total))
        random.Random(seed).shuffle(order)
        self.table = np.full((S, self.cols), -1, np.int32)
        at = 0
        for s in range(S):
            self.table[s, :self.old[s]] = order[at:at + self.old[s]]
            at += self.old[s]
        self.stack = np.zeros(self.total, np.int32)
        self.stack[:free] = order[at:]
        self.free = free
        self.tokens = sum(max(0, b - a) for a, b in zip(self.have, self.want))
        self.back = sum(max(0, a - b) for a, b in zip(self.have, self.want))  # tokens of the way back
        self.taken, self.given = taken, given


def _positions(c):
    """Positions of the tokens: a run for each of a few sequences, the last up to `far`."""
    rng = _rng(c)
    T = c["tokens"]
    cuts = sorted({0, T, *(rng.randrange(T + 1) for _ in range(min(T - 1, 4) if T < 256 else 3))})
    out = np.zeros(T, np.int32)
    if T <= 64:  # single tokens of many sequences
        out[:] = [rng.randrange(c["far"]) for _ in range(T)]
        out[-1] = c["far"] - 1
        return out
    for a, b in zip(cuts, cuts[1:]):
        out[a:b] = np.arange(b - a) + rng.randrange(max(1, c["far"] - (b - a)))
    return out


def _cache_slots(c):
    """Slots of the tokens, runs in pages that lie anywhere, and the cache's pages."""
    rng = _rng(dict(c, what="slots"))
    pages = -(-c["tokens"] // c["page"]) + 3
    order = list(range(pages))
    rng.shuffle(order)
    p = np.arange(c["tokens"]) + (rng.randrange(c["page"]) if c["tokens"] > 1 else 0)
    if c["tokens"] <= 64:  # a slot each in different pages
        pages, order = c["tokens"] + 3, list(range(c["tokens"] + 3))
        rng.shuffle(order)
        return np.array([order[i] * c["page"] + rng.randrange(c["page"]) for i in range(c["tokens"])], np.int32), pages
    return (np.array(order, np.int64)[p // c["page"]] * c["page"] + p % c["page"]).astype(np.int32), pages


def work(case):
    c = case
    if c["op"] == "pages":
        h = _Held(c, 0)
        # lengths in and out and starts, each page that moves read and written, a slot and a position a token; and back
        return {"bytes": 2 * (16.0 * c["seqs"] + 8.0 * (h.taken + h.given)) + 8.0 * (h.tokens + h.back), "flops": 0}
    if c["op"] in ("rotate", "store"):
        T, q, k = c["tokens"], c["heads"] * c["dim"], c["kv_heads"] * c["dim"]
        per = sum(k / 32 * (34 if t == "q8_0" else 18) for t in (c["k"], c["v"])) if c["op"] == "store" else 0
        moved = 8.0 * q + (8.0 * k if not per else 16.0 * k + 2 * per)  # store: k and v in, blocks out, blocks in, k and v out
        return {"bytes": T * (moved + 4), "flops": T * (q + k) * 7.0}
    T, N, K = c["tokens"], c["rows"], c["cols"]
    both = 2 if c["op"] == "gated" else 1
    return {"bytes": 4.0 * T * K + both * N * (K + 4.0) + 4.0 * T * N, "flops": 2.0 * both * T * N * K}


# -------------------------------------------------------------- operands
def _normal(shape, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)


def _i32(a):
    return torch.as_tensor(a, dtype=torch.int32, device=DEV)


def _qkv(c, seed):
    """q, k, v as views of one projection's output, [tokens, heads, dim], a few channels five times larger."""
    hq, hk, d = c["heads"], c["kv_heads"], c["dim"]
    x = _normal((c["tokens"], (hq + 2 * hk) * d), seed * 1000)
    x[:, 5::48] *= 5.0
    cut = lambda a, n: x[:, a * d:(a + n) * d].unflatten(1, (n, d))  # noqa: E731
    return cut(0, hq), cut(hq, hk), cut(hq + hk, hk)


def _weights(c, seed):
    """Norm weights of q and k."""
    if c["norm"] == "none":
        return None, None
    shape = lambda n: (n, c["dim"]) if c["norm"] == "heads" else (c["dim"],)  # noqa: E731
    return tuple(1.0 + 0.3 * _normal(shape(n), seed * 1000 + 1 + i) for i, n in enumerate((c["heads"], c["kv_heads"])))


def _freqs(c):
    """Radians a position of each pair, in 64 bits."""
    return 10000.0 ** (-2.0 * torch.arange(c["rotated"] // 2, dtype=torch.float64) / c["rotated"])


def _activations(c, seed):
    x = _normal((c["tokens"], c["cols"] + c["wide"]), seed * 1000)
    x[:, 7::96] *= 8.0
    return x[:, :c["cols"]]


def _matrix(c, seed, i):
    return _normal((c["rows"], c["cols"]), seed * 1000 + 1 + i) * c["cols"] ** -0.5


def _rows8(x):
    """int8 values as f32 and f32 scales of the rows of x. (Divisors are tensors: divided by, not multiplied with a reciprocal.)"""
    m = x.abs().amax(-1, keepdim=True)
    full = torch.full((), 127.0, device=x.device)
    r = torch.where(m >= 2.0 ** -100, full / m, torch.zeros_like(m))
    return (x * r).round_().clamp_(-127, 127), torch.where(m >= 2.0 ** -100, m / full, torch.zeros_like(m))


def _blocks(x, bits):
    """What the blocks of 32 of x [..., D] stand for in the cache."""
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    hi, lo = b.amax(-1), b.amin(-1)
    of = lambda v: torch.full((), v, device=x.device)  # noqa: E731
    d = torch.maximum(hi, -lo) / of(127.0) if bits == 8 else torch.where(hi >= -lo, hi, lo) / of(-8.0)
    f = d.half().float()
    r = torch.where(f != 0, of(1.0) / f, torch.zeros_like(f))
    q = (b * r[..., None]).round_().clamp_(*((-127, 127) if bits == 8 else (-8, 7)))
    return q.mul_(f[..., None]).reshape(x.shape)


def _bits(t):
    return 8 if t == "q8_0" else 4


# ------------------------------------------------------------------ cases
def prepare(case, seed):
    c, op = case, case["op"]
    s = {"case": c, "own": own}
    if own:
        import vortx_amd as vx
        quant = {"q4_0": vx.VX_Q4_0, "q8_0": vx.VX_Q8_0}
    if op == "pages":
        h = s["held"] = _Held(c, seed)
        s["want"], s["have"] = _i32(h.want), _i32(h.have)
        most = max(h.tokens, h.back, 1)
        if own:
            s["ops"] = vx.KvAttention(0)
            s["pages"] = vx.KvPages(h.total, c["page"], c["seqs"], h.cols, device=DEV)
            s["pages"].table.copy_(_i32(h.table))
            s["pages"].lens.copy_(s["have"])
            s["pages"].free.copy_(_i32(h.stack))
            s["pages"].free_count.fill_(h.free)
            s["step"], s["undo"] = vx.KvStep(c["seqs"], most, device=DEV), vx.KvStep(c["seqs"], most, device=DEV)
        else:
            s.update(table=_i32(h.table), lens=_i32(h.have), free=_i32(h.stack), count=_i32([h.free]), most=most)
        return s
    if op in ("rotate", "store"):
        s["q"], s["k"], s["v"] = _qkv(c, seed)
        s["wq"], s["wk"] = _weights(c, seed)
        s["freqs"], s["positions"] = _freqs(c).to(DEV), _i32(_positions(c))
        s["qo"], s["ko"] = (torch.empty_like(t, memory_format=torch.contiguous_format) for t in (s["q"], s["k"]))
        if own:
            s["ops"] = vx.KvAttention(0)
            s["how"] = s["ops"].rotation(s["freqs"], pairs=c["style"] == "pairs", norm=c["norm"] != "none", q_weight=s["wq"],
                                         k_weight=s["wk"], eps=EPS)
        if op == "store":
            at, pages = _cache_slots(c)
            s["slots"], s["vo"] = _i32(at), torch.empty_like(s["ko"])
            if own:
                s["cache"] = vx.KvCache(pages, c["page"], c["kv_heads"], c["dim"], quant[c["k"]], quant[c["v"]], device=DEV)
        return s
    s["x"] = _activations(c, seed)
    names = ("gate", "up") if op == "gated" else ("w",)
    if own:
        s["ops"] = vx.Int8Gemm(0)
        for i, n in enumerate(names):  # weights are laid out once
            s[n] = vx.Int8Rows.empty(c["rows"], c["cols"], device=DEV)
            s["ops"].quantize(s[n], _matrix(c, seed, i))
        s["out"] = torch.empty(c["tokens"], c["rows"], device=DEV)
        s["ws"] = vx.Int8Gemm.workspace(c["tokens"], c["cols"], device=DEV)
    else:
        for i, n in enumerate(names):
            q, d = _rows8(_matrix(c, seed, i))
            s[n], s[n + "_scale"] = q.to(torch.int8), d.squeeze(-1)
    return s


def _plain_step(s, want, most):
    """The pages that sequences give back and take, in the state's own buffers; starts, slots and positions of `most` tokens."""
    c, h = s["case"], s["held"]
    table, lens, free, count, page = s["table"], s["lens"], s["free"], s["count"], c["page"]
    up = lambda n: torch.div(n + page - 1, page, rounding_mode="floor")  # noqa: E731
    have = lens.clone()
    old, new = up(have), up(want)
    # given back: the last page of the last sequence first, so that taking them again finds them as they were
    gives = (old - new).clamp_min(0)
    ends = gives.cumsum(0)
    item = torch.arange(max(h.given, h.taken, 1), device=DEV)
    owner = torch.searchsorted(ends, item, right=True).clamp_max(c["seqs"] - 1)
    given = ends[-1]
    page_of = table[owner, (new[owner] + item - (ends - gives)[owner]).clamp(0, h.cols - 1)]
    free[torch.where(item < given, count + given - 1 - item, h.total)] = page_of
    total = count + given
    # taken: from the top, by the sequences that find all they need
    needs = (new - old).clamp_min(0)
    ends = needs.cumsum(0)
    served = (needs == 0) | (ends <= total)
    takes = torch.where(served, needs, 0)
    tends = takes.cumsum(0)
    owner = torch.searchsorted(tends, item, right=True).clamp_max(c["seqs"] - 1)
    there = item < tends[-1]
    got = free[(total - 1 - item).clamp_min(0)]
    row = torch.where(there, owner, c["seqs"])
    table[row, torch.where(there, old[owner] + item - (tends - takes)[owner], 0)] = got
    count.copy_(total - tends[-1])
    lens.copy_(torch.where(served, want, have))
    # the tokens that are new
    n = (want - have).clamp_min(0)
    starts = torch.zeros(c["seqs"] + 1, dtype=torch.int32, device=DEV)
    starts[1:] = n.cumsum(0)
    token = torch.arange(most, device=DEV, dtype=torch.int32)
    owner = torch.searchsorted(starts[1:], token, right=True).clamp_max(c["seqs"] - 1)
    live = token < starts[-1]
    pos = torch.where(live, have[owner] + token - starts[owner], 0)
    at = table[owner, torch.div(pos, page, rounding_mode="floor").clamp_max(h.cols - 1)] * page + pos % page
    return starts, torch.where(live & served[owner], at, -1), pos


def _plain_rotated(s, x, w, dtype):
    c = s["case"]
    x = x.to(dtype)
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.to(dtype)
    angle = s["positions"].double()[:, None] * s["freqs"]  # [T, pairs], in 64 bits: far positions
    cos, sin = angle.cos().to(dtype)[:, None], angle.sin().to(dtype)[:, None]
    turned, rest = x[..., :c["rotated"]], x[..., c["rotated"]:]
    if c["style"] == "pairs":
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turned.chunk(2, -1)
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, rest), -1).float()


def _plain_act(g, act):
    if act == "relu":
        return g.clamp_min(0)
    if act == "gelu":
        return 0.5 * g * torch.erfc(-g * 0.5 ** 0.5)
    if act == "gelu_tanh":
        return 0.5 * g * (1 + torch.tanh((2 / math.pi) ** 0.5 * (g + 0.044715 * g ** 3)))
    return g / (1 + torch.exp(-g))


def run(state):
    s, c = state, state["case"]
    op = c["op"]
    if op == "pages":
        if s["own"]:
            p, step = s["pages"], s["step"]
            s["ops"].resize(p, s["want"], step)
            s["ops"].resize(p, s["have"], s["undo"])
            return {"starts": step.starts, "slots": step.slots, "positions": step.positions, "table": p.table, "lens": p.lens,
                    "free": p.free, "count": p.free_count}
        # a row and a place more for what is not there
        table, free = s["table"], s["free"]
        s["table"] = torch.cat((table, table[:1]))
        s["free"] = torch.cat((free, free[:1]))
        starts, slots, pos = _plain_step(s, s["want"], s["most"])
        _plain_step(s, s["have"], s["most"])
        table.copy_(s["table"][:-1])
        free.copy_(s["free"][:-1])
        s["table"], s["free"] = table, free
        return {"starts": starts, "slots": slots, "positions": pos, "table": table, "lens": s["lens"], "free": free, "count": s["count"]}
    if op == "rotate":
        if s["own"]:
            s["ops"].rotate(s["qo"], s["q"], s["ko"], s["k"], s["positions"], s["how"])
            return s["qo"], s["ko"]
        return _plain_rotated(s, s["q"], s["wq"], torch.float32), _plain_rotated(s, s["k"], s["wk"], torch.float32)
    if op == "store":
        if s["own"]:
            s["ops"].write_rotated(s["cache"], s["qo"], s["q"], s["k"], s["v"], s["positions"], s["slots"], s["how"])
            s["ops"].read(s["ko"], s["vo"], s["cache"], s["slots"])
            return s["qo"], s["ko"], s["vo"]
        # k in 64 bits: in 32 some values come out on the other side of a border between two codes
        k = _plain_rotated(s, s["k"], s["wk"], torch.float64)
        return _plain_rotated(s, s["q"], s["wq"], torch.float32), _blocks(k, _bits(c["k"])), _blocks(s["v"], _bits(c["v"]))
    if s["own"]:
        if op == "gated":
            s["ops"].dispatch_gated(s["out"], s["x"], s["gate"], s["up"], act=c["act"], workspace=s["ws"])
        else:
            s["ops"].dispatch(s["out"], s["x"], s["w"], workspace=s["ws"])
        return s["out"]
    q, d = _rows8(s["x"])
    times = lambda n: torch.matmul(q, s[n].float().t()).mul_(d).mul_(s[n + "_scale"])  # noqa: E731
    return _plain_act(times("gate"), c["act"]) * times("up") if op == "gated" else times("w")


# ------------------------------------------------------------------ in 64 bits
def _f32(t):
    return t.float().double()


def _exact_rows8(x):
    x = x.double()
    m = x.abs().max(-1, keepdim=True).values
    small = m < 2.0 ** -100
    safe = torch.where(small, 1.0, m)
    q = torch.round(_f32(x * _f32(127 / safe))).clamp(-127, 127)
    return torch.where(small, 0.0, q), torch.where(small, 0.0, _f32(safe / 127))


def _exact_blocks(x, bits):
    b = x.double().reshape(*x.shape[:-1], -1, 32)
    top, low = b.max(-1).values, b.min(-1).values
    if bits == 8:
        d = _f32(torch.where(top > -low, top, -low) / 127)
    else:
        d = _f32(torch.where(-low > top, low, top) / -8)
    d = d.half().double()
    r = _f32(1 / torch.where(d == 0, 1.0, d)) * (d != 0)
    q = torch.round(_f32(b * r[..., None]))
    q = q.clamp(-127, 127) if bits == 8 else q.clamp(-8, 7)
    return (q * d[..., None]).reshape(x.shape)


def _exact_rotated(c, x, w):
    x = x.double()
    if w is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * w.double()
    turn = torch.as_tensor(_positions(c), device=DEV).double()[:, None, None] * _freqs(c).to(DEV)
    half = c["rotated"] // 2
    i = torch.arange(half, device=DEV)
    first, second = (2 * i, 2 * i + 1) if c["style"] == "pairs" else (i, i + half)
    z = torch.complex(x[..., first], x[..., second]) * torch.polar(torch.ones_like(turn), turn)
    out = x.clone()
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _exact_pages(c, seed):
    h = _Held(c, seed)
    stack, table, lens = [int(p) for p in h.stack[:h.free]], h.table.copy(), list(h.have)
    memory = h.stack.copy()

    def step(want):
        have = list(lens)
        need = lambda n: -(-n // c["page"])  # noqa: E731
        for s in reversed(range(c["seqs"])):
            for j in reversed(range(need(want[s]), need(have[s]))):
                memory[len(stack)] = table[s, j]
                stack.append(int(table[s, j]))
        room, asked, starts, slots, pos = len(stack), 0, [0], [], []
        for s in range(c["seqs"]):
            more = max(0, need(want[s]) - need(have[s]))
            asked += more
            fits = more == 0 or asked <= room
            if fits:
                for j in range(need(have[s]), need(want[s])):
                    table[s, j] = stack.pop()
                lens[s] = want[s]
            for p in range(have[s], want[s]):
                pos.append(p)
                slots.append(int(table[s, p // c["page"]]) * c["page"] + p % c["page"] if fits else -1)
            starts.append(len(pos))
        return starts, slots, pos

    starts, slots, pos = step(h.want)
    step(h.have)
    most = max(h.tokens, h.back, 1)
    pad = lambda a, v: _i32(a + [v] * (most - len(a)))  # noqa: E731
    return {"starts": _i32(starts), "slots": pad(slots, -1), "positions": pad(pos, 0), "table": _i32(table), "lens": _i32(lens),
            "free": _i32(memory), "count": _i32([len(stack)])}


def exact(case, seed):
    c, op = case, case["op"]
    if op == "pages":
        return _exact_pages(c, seed)
    if op in ("rotate", "store"):
        (q, k, v), (wq, wk) = _qkv(c, seed), _weights(c, seed)
        qo, ko = _exact_rotated(c, q, wq), _exact_rotated(c, k, wk)
        if op == "rotate":
            return qo, ko
        return qo, _exact_blocks(ko.float(), _bits(c["k"])), _exact_blocks(v, _bits(c["v"]))
    x, d = _exact_rows8(_activations(c, seed))

    def times(i):
        w, e = _exact_rows8(_matrix(c, seed, i))
        return (x @ w.t()) * d * e.squeeze(-1)

    if op == "product":
        return times(0)
    g = times(0)
    if c["act"] == "relu":
        g = torch.where(g > 0, g, 0.0)
    elif c["act"] == "gelu":
        g = g * torch.special.ndtr(g)
    elif c["act"] == "gelu_tanh":
        g = g * torch.sigmoid(math.sqrt(8 / math.pi) * (g + 0.044715 * g ** 3))
    else:
        g = g * torch.sigmoid(g)
    return g * times(1)
