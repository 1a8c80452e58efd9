"""A serving loop's decoder: sequences come, grow and go; pages, rotation, attention
and the feed-forward block all run on the device.

Pages of the cache are dealt out by :meth:`vortx_amd.KvAttention.resize`, queries and
keys normed and rotated by position on their way (:meth:`write_rotated`), attention
runs over the paged cache, and the projections and the gated feed-forward block are
products of 8-bit integers (:class:`vortx_amd.Int8Gemm`). A decode step has the same
calls and buffers every time, so it is captured once and replayed. Weights are
random: the point is the calls, and that single tokens, replayed, give what a prompt
of the same tokens gives.

    python examples/serve.py
"""
from __future__ import annotations

import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

import vortx_amd as vx  # noqa: E402

HIDDEN, HEADS, KV_HEADS, DIM, INNER, LAYERS, VOCAB, PAGE = 512, 8, 2, 64, 1408, 2, 1000, 16
DEV = "cuda:0"


class Server:
    def __init__(self, sequences: int, max_len: int, seed: int = 0):
        self.kv, self.i8 = vx.KvAttention(0), vx.Int8Gemm(0)
        g = torch.Generator(device=DEV).manual_seed(seed)
        normal = lambda *shape: torch.randn(*shape, generator=g, device=DEV)  # noqa: E731
        shapes = {"qkv": ((HEADS + 2 * KV_HEADS) * DIM, HIDDEN), "out": (HIDDEN, HEADS * DIM), "gate": (INNER, HIDDEN),
                  "up": (INNER, HIDDEN), "down": (HIDDEN, INNER)}
        self.weights = [{n: self._weight(normal(*s) * s[1] ** -0.5) for n, s in shapes.items()} for _ in range(LAYERS)]
        self.head = self._weight(normal(VOCAB, HIDDEN) * HIDDEN ** -0.5)
        self.embedding = normal(VOCAB, HIDDEN)
        self.how = [self.kv.rotation(vx.rotation_freqs(DIM), norm=True, q_weight=1 + 0.1 * normal(DIM), k_weight=1 + 0.1 * normal(DIM))
                    for _ in range(LAYERS)]
        cols = -(-max_len // PAGE)
        self.pages = vx.KvPages(sequences * cols, PAGE, sequences, cols)  # all layers use the same pages
        self.caches = [vx.KvCache(sequences * cols, PAGE, KV_HEADS, DIM, vx.VX_Q8_0, vx.VX_Q8_0) for _ in range(LAYERS)]
        self.max_len = max_len

    def _weight(self, w):
        rows = vx.Int8Rows.empty(*w.shape)
        self.i8.quantize(rows, w)
        return rows

    def buffers(self, tokens: int, queries: int):
        """What a step of up to so many tokens, `queries` of a sequence, works in."""
        b = {"step": vx.KvStep(self.pages.seqs, tokens), "want": torch.zeros(self.pages.seqs, dtype=torch.int32, device=DEV),
             "tokens": torch.zeros(tokens, dtype=torch.int64, device=DEV), "ws": vx.Int8Gemm.workspace(tokens, max(HIDDEN, INNER))}
        b["plans"] = [self.kv.plan(c, self.pages.table, self.pages.lens, b["step"].starts, q_heads=HEADS, max_queries=queries,
                                   max_len=self.max_len, tokens=tokens) for c in self.caches]
        empty = lambda *shape: torch.zeros(*shape, device=DEV)  # noqa: E731
        b.update(qkv=empty(tokens, (HEADS + 2 * KV_HEADS) * DIM), o=empty(tokens, HEADS, DIM), h=empty(tokens, HIDDEN),
                 inner=empty(tokens, INNER), logits=empty(tokens, VOCAB))
        return b

    def step(self, b):
        """Logits of b's tokens, whose sequences are brought to b's lengths."""
        step, ws = b["step"], b["ws"]
        self.kv.resize(self.pages, b["want"], step)
        x = self.embedding[b["tokens"]]
        norm = lambda t: torch.nn.functional.rms_norm(t, (HIDDEN,))  # noqa: E731
        q, k, v = (b["qkv"][:, i * DIM:j * DIM].unflatten(1, (-1, DIM)) for i, j in
                   ((0, HEADS), (HEADS, HEADS + KV_HEADS), (HEADS + KV_HEADS, HEADS + 2 * KV_HEADS)))
        for w, cache, plan, how in zip(self.weights, self.caches, b["plans"], self.how):
            self.i8.dispatch(b["qkv"], norm(x), w["qkv"], workspace=ws)
            self.kv.write_rotated(cache, q, q, k, v, step.positions, step.slots, how)
            self.kv.attend(b["o"], q, plan)
            self.i8.dispatch(b["h"], b["o"].flatten(1), w["out"], workspace=ws)
            x = x + b["h"]
            self.i8.dispatch_gated(b["inner"], norm(x), w["gate"], w["up"], "silu", workspace=ws)
            self.i8.dispatch(b["h"], b["inner"], w["down"], workspace=ws)
            x = x + b["h"]
        self.i8.dispatch(b["logits"], norm(x), self.head, workspace=ws)
        return b["logits"]


def main(sequences: int = 5, most: int = 45, generate: int = 7) -> float:
    """The largest difference between logits of tokens one by one and of the same as prompts, relative."""
    server = Server(sequences, most + generate + 3)
    g = torch.Generator().manual_seed(7)
    lengths = [int(torch.randint(1, most + 1, (1,), generator=g)) for _ in range(sequences)]
    texts = [torch.randint(VOCAB, (n + generate,), generator=g).to(DEV) for n in lengths]
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=DEV)  # noqa: E731

    prompts = server.buffers(sum(lengths) + sequences * generate, most + generate)
    prompts["tokens"][:sum(lengths)] = torch.cat([t[:n] for t, n in zip(texts, lengths)])
    prompts["want"].copy_(i32(lengths))
    server.step(prompts)
    one = server.buffers(sequences, 1)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    one["want"].copy_(server.pages.lens)  # (a step without new tokens, so that all code is there before the capture)
    server.step(one)
    with torch.cuda.graph(graph, stream=stream):
        server.step(one)
    single = []
    for i in range(generate):  # tokens one by one, all sequences together: the same graph each time
        one["want"].copy_(i32([n + i + 1 for n in lengths]))
        one["tokens"].copy_(torch.stack([t[n + i] for t, n in zip(texts, lengths)]))
        graph.replay()
        single.append(one["logits"].clone())
    # all sequences end and come back as prompts of all their tokens, in other pages
    prompts["want"].zero_()
    server.step(prompts)
    assert int(server.pages.free_count) == server.pages.pages
    prompts["want"].copy_(i32([n + generate for n in lengths]))
    prompts["tokens"].copy_(torch.cat(texts))
    logits, starts = server.step(prompts), prompts["step"].starts.tolist()
    again = torch.stack([logits[e - generate:e] for e in starts[1:]], 1)
    off = ((again - torch.stack(single)).abs().max() / again.abs().max()).item()
    print(f"{sequences} sequences of {min(lengths)} to {max(lengths)} tokens and {generate} more: logits off by {off:.2g}, relative")
    return off


if __name__ == "__main__":
    main()
