"""The gated product where its gates are as large and as small as f32 has them."""
import math

import numpy as np
import pytest
import torch

import vortx_amd as vx
from tests.helpers import note

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
UNIT = 2.0 ** -24  # half a step of f32, relative

SIZES = [3e38, 2.7e38, 2.4e38, 2.3e38, 1e30, 1e20, 1.6e13, 1.4e13, 1e6, 300, 126.5, 126, 104, 103, 100, 95, 92, 90, 89, 88.8, 88.5, 88, 87, 80, 60, 44.5, 44,
         20, 10.5, 9, 5, 1, 0.1, 1e-3, 1e-20, 1e-37, 1e-42]
GATES = np.array([s * v for v in SIZES for s in (1.0, -1.0)] + [0.0, math.inf, -math.inf], np.float64)


def _sigmoid(y):
    t = np.exp(-np.abs(y))
    return np.where(y >= 0, 1 / (1 + t), t / (1 + t))


def _times(g, s):
    return np.where(s == 0, 0.0, np.where(s == 0, 1.0, g) * s)  # (far below zero the sigmoid is nothing, whatever it is multiplied with)


def _tanh_y(g):
    return math.sqrt(8 / math.pi) * (g + 0.044715 * g ** 3)


def _erfc(z):
    return torch.erfc(torch.tensor(z, dtype=torch.float64)).numpy()


# Value of a gate g that is exact here; then the bound of its error in half steps, relative; then what is added where f32 has
# no normal numbers left, in numbers of 2^-149.
# The sigmoid: e^-y to 3 (the instruction's step, two of them, and a rounding), of which at most all reaches 1 + e^-y, 1 its sum, 1 the
# reciprocal after its Newton step; the product with g 1. y of the tanh form: two constants, three products and a sum, 6, which
# count |y| (1 - sigmoid(y)) times. erfc: 16 steps to the device's function, 32; its argument, 2 off, counts at most g^2 + 2 times; a
# product; erfc below f32's normal numbers may be 0, 2^-126 |g|. Numbers below the normal ones are rounded to 2^-150 once in the
# activation (where it is the end of a chain of relative errors) and once after the product with u.
ACTS = {
    "silu": (lambda g: _times(g, _sigmoid(g)), lambda g: 6 + 0 * g, lambda g: 1 + 0 * g),
    "gelu_tanh": (lambda g: _times(g, _sigmoid(_tanh_y(g))), lambda g: 6 + 6 * np.where(g > 0, 1.0, np.minimum(np.abs(_tanh_y(g)), 1e6)), lambda g: 1 + 0 * g),
    "gelu": (lambda g: _times(g, 0.5 * _erfc(-g / math.sqrt(2))), lambda g: 33 + 2 * (np.minimum(np.abs(g), 1e3) ** 2 + 2),
             lambda g: 1 + 2.0 ** 23 * np.minimum(np.abs(g), 1e3)),
    "relu": (lambda g: np.maximum(g, 0.0), lambda g: 0 * g, lambda g: 0 * g),
}


def _rows(codes, scales):
    rows, cols = codes.shape
    data = torch.full((rows, -(-cols // 16) * 16), 55, dtype=torch.int8, device=DEV)
    data[:, :cols] = torch.tensor(codes, device=DEV)
    return vx.Int8Rows(data, torch.tensor(np.asarray(scales, np.float32), device=DEV), cols)


@pytest.fixture(scope="module")
def i8():
    assert torch.cuda.is_available()
    return vx.Int8Gemm(0)


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("T,N,K,f32", [(1, 150, 64, True), (2, 150, 4096, True), (4, 150, 100, True),  # streamed
                                       (3, 150, 64, False), (30, 150, 128, False), (60, 800, 64, False),  # straight from memory
                                       (300, 1500, 65, False), (2049, 2100, 70, False),                  # tiles
                                       (100, 150, 2048, True), (130, 150, 4099, True)])                  # parts of K
def test_gates_of_any_size(i8, act, T, N, K, f32):
    """Codes of 127 and 1 in one column: a gate is 127 w sx, one rounding of it, which the oracle makes too."""
    note(f"gates {act} {T} x {N} x {K}")
    want = np.resize(GATES, N)
    with np.errstate(over="ignore"):
        scale = (want / 127).astype(np.float32)
    sx = (2.0 ** -(np.arange(T) % 3)).astype(np.float32)
    at = K - 1
    wc = np.zeros((N, K), np.int8)
    wc[:, at] = 1
    gate, up = _rows(wc, scale), _rows(wc, np.full(N, 2.0 ** -7, np.float32))
    with np.errstate(over="ignore", invalid="ignore", under="ignore"):
        # (a power of two before the rounding, as after it, but for numbers below the normal ones: rounded once from 64 bits)
        g = (127.0 * scale.astype(np.float64) * sx.astype(np.float64)[:, None])
        normal = np.abs(g) >= 2.0 ** -126
        g = np.where(normal, g.astype(np.float32), g).astype(np.float64)
        u = 127 * 2.0 ** -7 * sx.astype(np.float64)[:, None]
        value, bound, small = ACTS[act]
        a = value(g)
        ref = a * u
        # a gate below the normal numbers is itself rounded, to half of 2^-149; act'(g) is at most 1.13
        tol = np.abs(ref) * (bound(g) + 1) * 1.001 * UNIT + 2.0 ** -149 * (1 + (small(g) + 1) * u)
        tol = np.where(np.abs(ref) < np.inf, tol, 0)
    out = torch.full((T, N), float("nan"), device=DEV)
    if f32:
        x = torch.zeros(T, K, device=DEV)
        x[:, at] = 127 * torch.tensor(sx, device=DEV)
        i8.dispatch_gated(out, x, gate, up, act, workspace=i8.workspace(T, K))
    else:
        xc = np.zeros((T, K), np.int8)
        xc[:, at] = 127
        i8.dispatch_gated(out, _rows(xc, sx), gate, up, act)
    got = out.cpu().numpy().astype(np.float64)
    big = np.abs(ref) > np.finfo(np.float32).max * (1 - 2.0 ** -20)  # (past f32, or next to its end: infinity is right too)
    with np.errstate(invalid="ignore"):
        ok = (got == ref) | (np.abs(got - ref) <= tol) | (big & (got == np.sign(ref) * np.inf))
    bad = np.argwhere(~ok)
    assert ok.all(), [(float(g[t, n]), float(got[t, n]), float(ref[t, n])) for t, n in bad[:8]]


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("T,f32", [(1, True), (20, False), (200, False)])
def test_gates_that_are_no_numbers(i8, act, T, f32):
    """They and no other column become NaN."""
    K, N = 64, 90
    wc = np.zeros((N, K), np.int8)
    wc[:, 0] = 1
    scale = np.full(N, 0.01, np.float32)
    clean = scale.copy()
    scale[[3, 50]] = np.nan
    xc = np.zeros((T, K), np.int8)
    xc[:, 0] = 127
    outs = [torch.empty(T, N, device=DEV) for _ in range(2)]
    x = torch.tensor(xc, device=DEV).float() if f32 else _rows(xc, np.ones(T, np.float32))
    for o, s in zip(outs, (scale, clean)):
        i8.dispatch_gated(o, x, _rows(wc, s), _rows(wc, clean), act)
    keep = [n for n in range(N) if n not in (3, 50)]
    assert outs[0][:, [3, 50]].isnan().all() and torch.equal(outs[0][:, keep], outs[1][:, keep])
