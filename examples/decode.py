"""A small decoder on quantized weights and a quantized cache, as a serving loop
runs it: a prompt, tokens one by one, then drafts of several tokens checked at
once as a tree.

Projections are products with Q4_0 weights (:class:`vortx_amd.QuantGemv`), keys
and values go into a paged Q8_0 / Q4_0 cache and attention runs over it
(:class:`vortx_amd.KvAttention`); positions enter by a bias that grows with
distance. Weights are random: the point is the calls, and that a tree's logits
are those of its tokens taken one by one.

    python examples/decode.py
"""
from __future__ import annotations

import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

import vortx_amd as vx  # noqa: E402
from vortx_amd import synthetic  # noqa: E402

HIDDEN, HEADS, KV_HEADS, DIM, LAYERS, VOCAB, PAGE = 512, 8, 2, 64, 2, 1000, 16
DEV = "cuda:0"


class Decoder:
    def __init__(self, sequences: int, max_len: int, seed: int = 0):
        self.gemv, self.kv = vx.QuantGemv(0), vx.KvAttention(0)
        self.weights, self.caches = [], []
        pages = sequences * -(-max_len // PAGE)
        for layer in range(LAYERS):
            rows = {"q": HEADS * DIM, "k": KV_HEADS * DIM, "v": KV_HEADS * DIM, "out": HIDDEN}
            self.weights.append({n: self._weight(r, HIDDEN, seed + 10 * layer + i) for i, (n, r) in enumerate(rows.items())})
            self.caches.append(vx.KvCache(pages, PAGE, KV_HEADS, DIM, vx.VX_Q8_0, vx.VX_Q4_0))
        self.head = self._weight(VOCAB, HIDDEN, seed + 99)
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.embedding = torch.randn(VOCAB, HIDDEN, generator=g, device=DEV)
        self.slopes = torch.exp2(-torch.arange(1, HEADS + 1, device=DEV, dtype=torch.float32))
        # pages of a sequence lie anywhere in the caches; all layers use the same ones
        self.table = torch.randperm(pages, generator=g, device=DEV).to(torch.int32).reshape(sequences, -1)
        self.lens = torch.zeros(sequences, dtype=torch.int32, device=DEV)
        self.max_len = max_len

    @staticmethod
    def _weight(rows, cols, seed):
        return vx.QWeight(synthetic.quant_weights(vx.VX_Q4_0, rows, cols, seed, DEV), vx.VX_Q4_0, rows, cols)

    def _product(self, w, x):
        y = torch.empty(x.shape[0], w.rows, device=DEV)
        self.gemv.dispatch(y.t(), w, x.t(), workspace=vx.QuantGemv.workspace(w, x.shape[0]))
        return y

    def plans(self, queries: int):
        """A plan a layer, for steps of `queries` tokens of every sequence."""
        starts = torch.arange(len(self.lens) + 1, dtype=torch.int32, device=DEV) * queries
        return [self.kv.plan(c, self.table, self.lens, starts, q_heads=HEADS, max_queries=queries, max_len=self.max_len,
                             slopes=self.slopes) for c in self.caches]

    def step(self, tokens, plans, tree=None):
        """Logits of `tokens` [sequences, n], which go into the cache behind what
        is there. With `tree` ([sequences * n, words], vx.tree_mask) they are drafts."""
        n = tokens.shape[1]
        pos = self.lens[:, None] + torch.arange(n, device=DEV)
        slots = (self.table.gather(1, (pos // PAGE).long()) * PAGE + pos % PAGE).to(torch.int32).flatten()
        self.lens += n  # the plans read it on the device
        x = self.embedding[tokens.flatten()]
        for w, cache, plan in zip(self.weights, self.caches, plans):
            h = torch.nn.functional.rms_norm(x, (HIDDEN,))
            q, k, v = (self._product(w[i], h).unflatten(1, (-1, DIM)) for i in "qkv")
            self.kv.write(cache, k, v, slots)
            o = torch.empty_like(q)
            if tree is None:
                self.kv.attend(o, q, plan)
            else:
                self.kv.attend_tree(o, q, plan, tree)
            x = x + self._product(w["out"], o.flatten(1))
        return self._product(self.head, torch.nn.functional.rms_norm(x, (HIDDEN,))).unflatten(0, (-1, n))

    def forget(self, n: int):
        """Takes the last n tokens of every sequence back."""
        self.lens -= n


def main(sequences: int = 3, prompt: int = 41, generate: int = 4) -> float:
    """The largest difference between logits of a tree and of single tokens."""
    model = Decoder(sequences, prompt + generate + 16)
    tokens = torch.randint(VOCAB, (sequences, prompt), generator=torch.Generator(device=DEV).manual_seed(7), device=DEV)
    logits = model.step(tokens, model.plans(prompt))[:, -1]
    one = model.plans(1)
    taken, single = [], []
    for _ in range(generate):
        taken.append(logits.argmax(-1))
        logits = model.step(taken[-1][:, None], one)[:, 0]
        single.append(logits)
    # the same tokens as drafts, each with another one beside it that leads nowhere
    model.forget(generate)
    drafts, parents, path = [], [], []
    for i, t in enumerate(taken):
        parent = path[-1] if path else -1
        path.append(len(drafts))
        drafts += [t, (t + 1) % VOCAB]
        parents += [parent, parent]
    tree = vx.tree_mask([parents] * sequences)
    checked = model.step(torch.stack(drafts, 1), model.plans(len(drafts)), tree)[:, path]
    off = (checked - torch.stack(single, 1)).abs().max().item()
    accepted = (checked[:, :-1].argmax(-1) == torch.stack(taken[1:], 1)).long().cumprod(1).sum(1) + 1
    print(f"drafts accepted by sequence: {accepted.tolist()} of {generate}; logits off by {off:.2g} of {checked.abs().max().item():.3g}")
    return off / checked.abs().max().item()


if __name__ == "__main__":
    main()
