"""The quantized key/value cache and the attention over it, as measurable cases.

`listed()` names twelve cases and `draw()` gives more of the same ranges;
`prepare(case, seed)` makes what a program holds before a call, `run(state)` is
one pass, `exact(case, seed)` the same results in 64 bits and `work(case)` what
a pass cannot do without. With `own` false `run` is the plain form: elementary
torch operations in f32 on a cache of int8 values and f16 scales. With `own`
true it makes the calls of `vortx_amd.KvAttention` on a `vortx_amd.KvCache`,
which keeps the same values in its own layout (so `prepare` fills the one or
the other from the same keys and values).

Operators (T tokens in S sequences, H key/value heads of D values, G query
heads for each):

* store: K and V of T tokens are quantized into cache slots, then read back;
* fetch: the rows of T slots, as f32;
* attend: softmax(scale q k^T, capped, biased, masked) v over each sequence's
  cache, for single tokens, prompts and chunks of prompts;
* tree: the same for drafted tokens, each of which sees its ancestors.

Quantization of a block of 32 values x (along D): 8 bits, d = f16(max|x| / 127)
and q = clamp(rint(x (1 / d)), -127, 127); 4 bits, m the value of the largest
magnitude, d = f16(m / -8) and q = clamp(rint(x (1 / d)), -8, 7). It stands for
d q.
"""
from __future__ import annotations

import random

import numpy as np
import torch

own = False
DEV = "cuda:0"


# ----------------------------------------------------------------- cases
def _store(name, seqs, queries, history, heads, dim, page, k, v):
    return {"name": name, "op": "store", "seqs": seqs, "queries": queries, "history": history, "heads": heads, "dim": dim,
            "page": page, "k": k, "v": v}


def _fetch(name, seqs, history, heads, dim, page, k, v):
    return {"name": name, "op": "fetch", "seqs": seqs, "queries": 0, "history": history, "heads": heads, "dim": dim,
            "page": page, "k": k, "v": v}


def _attend(name, seqs, queries, history, heads, group, dim, page, k, v, op="attend", cap=0.0, slopes=False, window=0, docs=0,
            prefix=0):
    return {"name": name, "op": op, "seqs": seqs, "queries": queries, "history": history, "heads": heads, "group": group,
            "dim": dim, "page": page, "k": k, "v": v, "cap": cap, "slopes": slopes, "window": window, "docs": docs,
            "prefix": prefix}


def listed():
    return [
        # One token of each of five sequences goes into the cache in a decode step: the smallest call.
        _store("store_tokens", 5, 1, 900, 8, 128, 16, "q8_0", "q8_0"),
        # The keys and values of prompts of up to 4000 tokens, values in 4 bits.
        _store("store_prompts", 3, 4000, 0, 8, 128, 64, "q8_0", "q4_0"),
        # A short history read back, few heads of another size.
        _fetch("fetch_short", 1, 333, 3, 64, 16, "q4_0", "q8_0"),
        # Histories of several sequences read back, to be moved to another place or format.
        _fetch("fetch_histories", 4, 16000, 8, 128, 64, "q4_0", "q4_0"),
        # One decode step of one sequence: latency.
        _attend("decode_one", 1, 1, 777, 8, 4, 128, 16, "q8_0", "q8_0"),
        # One decode step of a serving batch, histories of all lengths.
        _attend("decode_batch", 32, 1, 8000, 8, 4, 128, 64, "q8_0", "q8_0"),
        # One decode step on a very long history, keys in 8 and values in 4 bits, scores capped.
        _attend("decode_long", 1, 1, 131000, 8, 8, 128, 256, "q8_0", "q4_0", cap=50.0),
        # A prompt, every query head with a key head of its own, scores capped.
        _attend("prompt", 1, 4096, 0, 32, 1, 128, 64, "q8_0", "q8_0", cap=30.0),
        # Prompts packed from several documents each, with a bias by distance and a window.
        _attend("prompt_documents", 3, 2500, 0, 4, 4, 64, 32, "q8_0", "q4_0", slopes=True, window=1000, docs=5),
        # A chunk of prompts whose first part sees all of itself, behind a history, in 4 bits.
        _attend("chunk_prefix", 4, 500, 3000, 8, 4, 128, 64, "q4_0", "q4_0", prefix=3100),
        # The drafts of one sequence checked at once: latency.
        _attend("tree_one", 1, 26, 1500, 8, 4, 128, 16, "q8_0", "q8_0", op="tree"),
        # The drafts of a batch.
        _attend("tree_batch", 8, 61, 12000, 8, 4, 128, 64, "q8_0", "q4_0", op="tree"),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["store", "fetch", "decode", "decode", "prompt", "prompt", "tree", "tree"])
    heads, dim, page = rng.choice([1, 2, 3, 4, 8, 8, 12, 16]), rng.choice([64, 96, 128, 128, 256]), rng.choice([16, 32, 64, 128, 256])
    k, v = rng.choice(["q8_0", "q4_0"]), rng.choice(["q8_0", "q4_0"])
    cost = lambda seqs, tokens: seqs * tokens * heads * dim  # noqa: E731
    if op in ("store", "fetch"):
        seqs, tokens = _log(rng, 1, 16), _log(rng, 1, 16000)
        while cost(seqs, tokens) > 6e7:
            tokens = tokens // 2 + 1
        c = _store("", seqs, tokens, rng.randint(0, 500), heads, dim, page, k, v) if op == "store" else \
            _fetch("", seqs, tokens, heads, dim, page, k, v)
    else:
        group = rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16])
        extra = dict(cap=rng.choice([0.0, 0.0, 30.0, 50.0]), slopes=rng.random() < 0.3)
        seqs, history = _log(rng, 1, 64), _log(rng, 1, 130000)
        if op == "decode":
            while cost(seqs, history) > 2.6e8:
                seqs, history = (seqs + 1) // 2, history // 2 + 1
            extra["window"] = rng.choice([0, 0, 0, _log(rng, 64, 8192)])
            c = _attend("", seqs, 1, history, heads, group, dim, page, k, v, **extra)
        elif op == "tree":
            queries = _log(rng, 2, 128)
            while cost(seqs, history) > 1.3e8 or cost(seqs, history) * group * queries > 2.5e10:
                seqs, history, queries = (seqs + 1) // 2, history // 2 + 1, queries // 2 + 1
            c = _attend("", seqs, queries, history, heads, group, dim, page, k, v, op="tree", **extra)
        else:
            seqs, queries, history = _log(rng, 1, 8), _log(rng, 2, 4096), rng.choice([0, 0, _log(rng, 1, 8192)])
            while cost(seqs, queries + history) * group * queries > 3.4e10:
                seqs, queries, history = (seqs + 1) // 2, queries * 2 // 3 + 1, history // 2
            extra["window"] = rng.choice([0, 0, _log(rng, 16, 4096)])
            extra["docs"] = rng.choice([0, 0, rng.randint(2, 9)])
            extra["prefix"] = rng.choice([0, 0, history + rng.randint(1, queries)])
            c = _attend("", seqs, queries, history, heads, group, dim, page, k, v, **extra)
    del c["name"]
    return c


# ------------------------------------------------ sizes that follow from a case
class _Sizes:
    """Lengths, positions, masks and pages, from the case alone."""

    def __init__(self, c):
        rng = random.Random(repr(sorted((k, v) for k, v in c.items() if k != "name")))
        ragged = lambda most: max(min(most, 1), int(most * rng.uniform(0.3, 1.0)))  # noqa: E731
        S = c["seqs"]
        self.n = [c["queries"]] + [ragged(c["queries"]) for _ in range(S - 1)]
        self.hist = [c["history"]] + [ragged(c["history"]) for _ in range(S - 1)]
        self.lens = [a + b for a, b in zip(self.n, self.hist)]
        self.starts = np.concatenate([[0], np.cumsum(self.n)]).astype(np.int32)
        self.T = int(self.starts[-1])
        need = [-(-L // c["page"]) for L in self.lens]
        self.pages, self.cols = sum(need) + 3, max(need)
        order = list(range(self.pages))
        rng.shuffle(order)  # pages are dealt out as they come free
        self.table = np.zeros((S, self.cols), np.int32)
        at = 0
        for s in range(S):
            self.table[s, :need[s]] = order[at:at + need[s]]
            at += need[s]
        self.first = self.prefix = self.parents = None
        if c.get("docs"):
            self.first = np.zeros(self.T, np.int32)
            for s in range(S):
                cuts = np.array(sorted([0] + [rng.randrange(self.lens[s]) for _ in range(c["docs"] - 1)]))
                pos = self.hist[s] + np.arange(self.n[s])
                self.first[self.starts[s]:self.starts[s + 1]] = cuts[np.searchsorted(cuts, pos, "right") - 1]
        if c.get("prefix"):
            self.prefix = np.array([min(c["prefix"], L) for L in self.lens], np.int32)
        if c["op"] == "tree":  # parents: mostly one of the last few drafts, now and then a root
            self.parents = [[rng.randint(max(-1, j - 6), j - 1) for j in range(n)] for n in self.n]

    def slots(self, c, s, lo, hi):
        """Cache slots of positions lo to hi of sequence s."""
        p = np.arange(lo, hi)
        return (self.table[s, p // c["page"]].astype(np.int64) * c["page"] + p % c["page"]).astype(np.int32)

    def sees(self, s):
        """Tree: [n, n], whether draft i sees draft j (an ancestor or itself)."""
        m = np.eye(self.n[s], dtype=bool)
        for j, p in enumerate(self.parents[s]):
            if p >= 0:
                m[j] |= m[p]
        return m

    def tree_words(self, c):
        words = -(-c["queries"] // 32)
        out = np.zeros((self.T, words), np.uint32)
        for s in range(c["seqs"]):
            m = np.zeros((self.n[s], words * 32), bool)
            m[:, :self.n[s]] = self.sees(s)
            out[self.starts[s]:self.starts[s + 1]] = np.packbits(m, axis=1, bitorder="little").view(np.uint32)
        return out.view(np.int32)

    def bounds(self, c, s):
        """First and last (exclusive) key in reach of each query of s, the drafts of a tree left out."""
        if c["op"] == "tree":
            pos = self.hist[s] + self.sees(s).sum(1) - 1
            hi = np.full(self.n[s], self.hist[s])
        else:
            pos = self.hist[s] + np.arange(self.n[s])
            hi = pos + 1
            if self.prefix is not None:
                hi = np.maximum(hi, self.prefix[s])
        lo = np.zeros(self.n[s], np.int64)
        if self.first is not None:
            lo = np.maximum(lo, self.first[self.starts[s]:self.starts[s + 1]])
        if c["window"]:
            lo = np.maximum(lo, pos - c["window"] + 1)
            hi = np.minimum(hi, pos + c["window"])
        return pos, lo, np.minimum(hi, self.lens[s])


def work(case):
    c, z = case, _Sizes(case)
    per = sum(c["heads"] * c["dim"] / 32 * (34 if t == "q8_0" else 18) for t in (c["k"], c["v"]))  # a token's K and V
    if c["op"] == "store":  # f32 in, blocks out, blocks in, f32 out
        return {"bytes": z.T * (16.0 * c["heads"] * c["dim"] + 2 * per), "flops": 0}
    if c["op"] == "fetch":
        return {"bytes": sum(z.lens) * (8.0 * c["heads"] * c["dim"] + per), "flops": 0}
    keys = pairs = 0
    for s in range(c["seqs"]):
        _, lo, hi = z.bounds(c, s)
        drafts = int(z.sees(s).sum()) if c["op"] == "tree" else 0
        pairs += int(np.maximum(hi - lo, 0).sum()) + drafts
        keys += max(0, int(hi.max() - lo.min())) + (z.n[s] if drafts else 0)
    hq = c["heads"] * c["group"]
    return {"bytes": keys * per + z.T * hq * c["dim"] * 8.0, "flops": 4.0 * pairs * hq * c["dim"]}


# -------------------------------------------------------------- operands
def _normal(shape, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)


def _keys_values(c, tokens, seed, s):
    """K and V [tokens, heads, dim] of sequence s: keys with a few channels five times larger, values normal."""
    k, v = (_normal((tokens, c["heads"], c["dim"]), seed * 1000 + 2 * s + i) for i in range(2))
    k[..., 5::48] *= 5.0
    return k, v


def _queries(c, z, seed):
    return _normal((z.T, c["heads"] * c["group"], c["dim"]), seed * 1000 + 999)


def _slopes(c):
    """2^(-8 (h + 1) / heads)."""
    n = c["heads"] * c["group"]
    return torch.exp2(-8.0 * torch.arange(1, n + 1, dtype=torch.float32) / n)


def _quantized(x, bits):
    """int8 values and f16 scales of the blocks of x [..., D]."""
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    hi, lo = b.amax(-1), b.amin(-1)
    of = lambda v: torch.full((), v, device=x.device)  # noqa: E731  (a tensor: divided by, not multiplied with its reciprocal)
    d = torch.maximum(hi, -lo) / of(127.0) if bits == 8 else torch.where(hi >= -lo, hi, lo) / of(-8.0)
    d = d.half()
    f = d.float()
    r = torch.where(f != 0, of(1.0) / f, torch.zeros_like(f))
    q = (b * r[..., None]).round_().clamp_(*((-127, 127) if bits == 8 else (-8, 7))).to(torch.int8)
    return q.reshape(x.shape), d


def _values(q, d):
    """What int8 values [..., D] and f16 scales [..., D / 32] stand for."""
    b = q.reshape(*q.shape[:-1], d.shape[-1], 32).float()
    return b.mul_(d.float()[..., None]).reshape(q.shape)


def _bits(t):
    return 8 if t == "q8_0" else 4


def _i32(a):
    return torch.as_tensor(a, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------ cases
def prepare(case, seed):
    c, z = case, _Sizes(case)
    s = {"case": c, "own": own}
    store = c["op"] == "store"
    if own:
        import vortx_amd as vx
        quant = {"q4_0": vx.VX_Q4_0, "q8_0": vx.VX_Q8_0}
        ops = s["ops"] = vx.KvAttention(0)
        cache = s["cache"] = vx.KvCache(z.pages, c["page"], c["heads"], c["dim"], quant[c["k"]], quant[c["v"]], device=DEV)
    else:
        shape = (z.pages * c["page"], c["heads"], c["dim"])
        for n in "kv":
            s[n + "q"] = torch.zeros(shape, dtype=torch.int8, device=DEV)
            s[n + "d"] = torch.zeros((*shape[:2], c["dim"] // 32), dtype=torch.float16, device=DEV)
    for i in range(0 if store else c["seqs"]):  # the histories (and, for attention, the queries' own keys) are in the cache
        k, v = _keys_values(c, z.lens[i], seed, i)
        at = _i32(z.slots(c, i, 0, z.lens[i]))
        if own:
            ops.write(cache, k, v, at)
        else:
            for n, x in (("k", k), ("v", v)):
                s[n + "q"][at.long()], s[n + "d"][at.long()] = _quantized(x, _bits(c[n]))
    if c["op"] in ("store", "fetch"):
        lo = z.hist if store else [0] * c["seqs"]
        s["slots"] = _i32(np.concatenate([z.slots(c, i, lo[i], z.lens[i]) for i in range(c["seqs"])]))
        if store:
            new = [_keys_values(c, z.n[i], seed, i) for i in range(c["seqs"])]
            s["k"], s["v"] = (torch.cat([x[i] for x in new]) for i in range(2))
        else:
            s["k"] = s["v"] = torch.empty((s["slots"].numel(), c["heads"], c["dim"]), device=DEV)
        s["ko"], s["vo"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
        return s
    # what a serving program keeps beside the cache: page table, lengths, starts, masks
    s["q"] = _queries(c, z, seed)
    s["out"] = torch.empty_like(s["q"])
    slopes = _slopes(c).to(DEV) if c["slopes"] else None
    tree = _i32(z.tree_words(c)) if c["op"] == "tree" else None
    s["tree"] = tree
    if own:
        s["plan"] = ops.plan(cache, _i32(z.table), _i32(z.lens), _i32(z.starts), q_heads=c["heads"] * c["group"],
                             max_queries=max(z.n), max_len=max(z.lens), softcap=c["cap"], slopes=slopes, window=c["window"],
                             first=None if z.first is None else _i32(z.first),
                             prefix=None if z.prefix is None else _i32(z.prefix))
        return s
    S, most = c["seqs"], max(z.n)
    row = np.zeros((S, most), np.int64)  # the token of each sequence's j-th query, and the bounds of what it sees
    pos, lo, hi = (np.zeros((S, most), np.int64) for _ in range(3))
    for i in range(S):
        row[i, :z.n[i]] = np.arange(z.starts[i], z.starts[i + 1])
        pos[i, :z.n[i]], lo[i, :z.n[i]], hi[i, :z.n[i]] = z.bounds(c, i)
    place = np.concatenate([i * most + np.arange(z.n[i]) for i in range(S)])
    up = lambda a: torch.as_tensor(a, device=DEV)  # noqa: E731
    s.update(row=up(row), pos=up(pos), lo=up(lo), hi=up(hi), place=up(place), slopes=slopes, hist=up(np.array(z.hist)),
             n=up(np.array(z.n)), keys=up(z.table.astype(np.int64))[:, :, None].mul(c["page"])
             .add(torch.arange(c["page"], device=DEV)).reshape(S, -1)[:, :max(z.lens)].contiguous())
    return s


def _plain_attention(s):
    c = s["case"]
    S, (T, Hq, D), H, G = c["seqs"], s["q"].shape, c["heads"], c["group"]
    keys, row = s["keys"], s["row"]
    L, N = keys.shape[1], row.shape[1]
    k = _values(s["kq"][keys], s["kd"][keys]).permute(0, 2, 3, 1).contiguous()  # [S, H, D, L]
    v = _values(s["vq"][keys], s["vd"][keys]).permute(0, 2, 1, 3).contiguous()  # [S, H, L, D]
    q = s["q"][row].mul_(D ** -0.5).reshape(S, N, H, G, D).permute(0, 2, 3, 1, 4).reshape(S, H, G * N, D)
    x = torch.matmul(q, k)
    if c["cap"]:
        x = x.div_(c["cap"]).tanh_().mul_(c["cap"])
    x = x.reshape(S, H, G, N, L)
    at = torch.arange(L, device=DEV)
    sees = (at >= s["lo"][..., None]) & (at < s["hi"][..., None])  # [S, N, L]
    where = at.expand(S, L)
    if s["tree"] is not None:  # drafted keys: where the query's bit is set, at the depth of the draft in its tree
        bits = (s["tree"][row][..., None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1  # [S, N, words, 32]
        bits = bits.reshape(S, N, -1)
        j = at - s["hist"][:, None]  # [S, L]
        draft = (j >= 0) & (j < s["n"][:, None])
        jj = j.clamp(0, N - 1)
        seen = bits.gather(2, jj[:, None, :].expand(S, N, L)) > 0
        depth = bits.sum(-1) - 1
        where = torch.where(draft, s["hist"][:, None] + depth.gather(1, jj), where)
        if c["window"]:
            seen &= (s["pos"][..., None] - where[:, None, :]).abs() < c["window"]
        sees = torch.where(draft[:, None, :], seen, sees)
    if c["slopes"]:
        far = (s["pos"][..., None] - where[:, None, :]).abs().float()
        x.sub_(s["slopes"].reshape(H, G, 1, 1) * far[:, None, None])
    x.masked_fill_(~sees[:, None, None], -float("inf"))
    x = x.sub_(x.amax(-1, keepdim=True).clamp_min_(-1e30)).exp_()  # a row that sees nothing: exp(-inf) = 0 throughout
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.reshape(S, H, G * N, L), v).reshape(S, H, G, N, D) / torch.where(total > 0, total, 1.0)
    return o.permute(0, 3, 1, 2, 4).reshape(S * N, Hq, D)[s["place"]]


def run(state):
    s, op = state, state["case"]["op"]
    if s["own"]:
        if op == "store":
            s["ops"].write(s["cache"], s["k"], s["v"], s["slots"])
        if op in ("store", "fetch"):
            s["ops"].read(s["ko"], s["vo"], s["cache"], s["slots"])
            return s["ko"], s["vo"]
        if op == "tree":
            s["ops"].attend_tree(s["out"], s["q"], s["plan"], s["tree"])
        else:
            s["ops"].attend(s["out"], s["q"], s["plan"])
        return s["out"]
    if op in ("store", "fetch"):
        c, at = s["case"], s["slots"].long()
        if op == "store":
            s["kq"][at], s["kd"][at] = _quantized(s["k"], _bits(c["k"]))
            s["vq"][at], s["vd"][at] = _quantized(s["v"], _bits(c["v"]))
        return _values(s["kq"][at], s["kd"][at]), _values(s["vq"][at], s["vd"][at])
    return _plain_attention(s)


def _exact_values(x, bits):
    """The values that the blocks of x [..., D] stand for, in 64 bits; f32 and f16 roundings where the definition has them."""
    f32 = lambda t: t.float().double()  # noqa: E731
    b = x.double().reshape(*x.shape[:-1], -1, 32)
    top, low = b.max(-1).values, b.min(-1).values
    if bits == 8:
        d = f32(torch.where(top > -low, top, -low) / 127)
    else:
        d = f32(torch.where(-low > top, low, top) / -8)
    d = d.half().double()
    r = f32(1 / torch.where(d == 0, 1.0, d)) * (d != 0)
    q = torch.round(f32(b * r[..., None]))
    q = q.clamp(-127, 127) if bits == 8 else q.clamp(-8, 7)
    return (q * d[..., None]).reshape(x.shape)


def exact(case, seed):
    c, z = case, _Sizes(case)
    if c["op"] in ("store", "fetch"):
        count = z.n if c["op"] == "store" else z.lens
        both = [[_exact_values(x, _bits(c[n])) for n, x in zip("kv", _keys_values(c, count[i], seed, i))] for i in range(c["seqs"])]
        return torch.cat([b[0] for b in both]), torch.cat([b[1] for b in both])
    q = _queries(c, z, seed).double()
    slopes = _slopes(c).double().to(DEV)
    out = torch.zeros_like(q)
    for s in range(c["seqs"]):
        k, v = _keys_values(c, z.lens[s], seed, s)
        k, v = _exact_values(k, _bits(c["k"])), _exact_values(v, _bits(c["v"]))
        pos, lo, hi = (torch.as_tensor(a, device=DEV) for a in z.bounds(c, s))
        at = torch.arange(z.lens[s], device=DEV)
        see = (at[None] >= lo[:, None]) & (at[None] < hi[:, None])
        where = at.clone()
        if c["op"] == "tree":
            where[z.hist[s]:] = pos
            see[:, z.hist[s]:] = torch.as_tensor(z.sees(s), device=DEV)
            if c["window"]:
                see[:, z.hist[s]:] &= (pos[:, None] - pos[None]).abs() < c["window"]
        rows = slice(int(z.starts[s]), int(z.starts[s + 1]))
        for h in range(c["heads"] * c["group"]):
            x = q[rows, h] @ k[:, h // c["group"]].t() / c["dim"] ** 0.5
            if c["cap"]:
                x = c["cap"] * torch.tanh(x / c["cap"])
            if c["slopes"]:
                x = x - slopes[h] * (pos[:, None] - where[None]).abs()
            x[~see] = -torch.inf
            x = torch.softmax(x, -1).nan_to_num(0.0)  # (a row that sees nothing)
            out[rows, h] = x @ v[:, h // c["group"]]
    return out
