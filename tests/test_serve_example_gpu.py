"""examples/serve.py: pages, rotation, attention, int8 products and gated blocks
together, single tokens from a replayed graph against prompts of the same tokens."""
import pytest

from tests.helpers import note

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sequences,most,generate", [(5, 45, 7), (1, 3, 2), (17, 20, 3)])
def test_serving_loop(sequences, most, generate):
    """The steps differ in f32 roundings only, but a value next to a border between two codes of an 8-bit row
    or block may take the other one, a step of 1 / 127 of the largest (through two layers, each with five
    products): a few steps at worst."""
    from examples import serve
    note(f"serve {sequences} sequences of up to {most}")
    assert serve.main(sequences, most, generate) < 4 / 127


def _plain(server, text):
    """Logits of a sequence in float64, from the weights' integers."""
    import torch
    from examples import serve as e
    f = lambda rows: rows.data[:, :rows.cols].double() * rows.scales[:, None].double()  # noqa: E731
    norm = lambda t, eps: t / (t.square().mean(-1, keepdim=True) + eps).sqrt()  # noqa: E731
    n, heads = len(text), e.HEADS + e.KV_HEADS
    angle = torch.arange(n, device=e.DEV).double()[:, None, None] * 10000.0 ** (-2 * torch.arange(e.DIM // 2, device=e.DEV).double() / e.DIM)
    x = server.embedding[text].double()
    eps32 = torch.finfo(torch.float32).eps
    for w, how in zip(server.weights, server.how):
        qkv = (norm(x, eps32) @ f(w["qkv"]).T).unflatten(1, (-1, e.DIM))
        _, q_weight, k_weight = how.keep
        weight = torch.cat([q_weight.double().expand(e.HEADS, -1), k_weight.double().expand(e.KV_HEADS, -1)])
        lo, hi = (norm(qkv[:, :heads], 1e-6) * weight).chunk(2, -1)
        qk = torch.cat([lo * angle.cos() - hi * angle.sin(), hi * angle.cos() + lo * angle.sin()], -1).transpose(0, 1)
        each = e.HEADS // e.KV_HEADS
        k, v = qk[e.HEADS:].repeat_interleave(each, 0), qkv[:, heads:].transpose(0, 1).repeat_interleave(each, 0)
        score = (qk[:e.HEADS, :, None] * k[:, None]).sum(-1) / e.DIM ** 0.5
        score = score.masked_fill(torch.ones(n, n, device=e.DEV).triu(1).bool(), float("-inf"))
        o = (score.softmax(-1)[..., None] * v[:, None]).sum(2).transpose(0, 1).flatten(1)
        x = x + o @ f(w["out"]).T
        y = norm(x, eps32)
        x = x + (torch.nn.functional.silu(y @ f(w["gate"]).T) * (y @ f(w["up"]).T)) @ f(w["down"]).T
    return norm(x, eps32) @ f(server.head).T


@pytest.mark.parametrize("lengths", [(9, 0, 1, 33), (1, 1, 1, 1), (40, 16, 17, 15)])
def test_serving_loop_against_float64(lengths):
    """The weights' integers are taken as they are, so what differs is the rounding of x to 8 bits, a step of
    max / 127: an error of max / 127 / sqrt(12) each, 0.8 % of x's root mean square at a largest of 3.5 of it and
    2.3 % at 10 (a gated product's). It comes five times a layer and once at the end, nine and two of them, and
    the cache's rounding is smaller than one; in root mean square they add to at most
    sqrt(9) 0.8 % + sqrt(2) 2.3 % < 6 %."""
    import torch
    from examples import serve as e
    note(f"serve {lengths} against float64")
    server = e.Server(len(lengths), 48, seed=3)
    b = server.buffers(sum(lengths) + 2, max(lengths))
    text = [torch.randint(e.VOCAB, (n,), device=e.DEV) for n in lengths]
    b["tokens"][:sum(lengths)] = torch.cat(text)
    b["want"].copy_(torch.tensor(lengths, dtype=torch.int32, device=e.DEV))
    logits = server.step(b)[:sum(lengths)].double()
    want = torch.cat([_plain(server, t) for t in text if len(t)])
    assert ((logits - want).square().mean() / want.square().mean()).sqrt().item() < 0.06
