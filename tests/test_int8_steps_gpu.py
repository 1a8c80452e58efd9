"""How far products of 8-bit integers are off, in f32's steps, with sums that f32
does not hold exactly."""
import numpy as np
import pytest
import torch

import vortx_amd as vx
from tests.helpers import note

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _rows(codes, scales):
    rows, cols = codes.shape
    data = torch.zeros(rows, -(-cols // 16) * 16, dtype=torch.int8, device=DEV)
    data[:, :cols] = torch.tensor(codes, device=DEV)
    return vx.Int8Rows(data, torch.tensor(scales, device=DEV), cols)


@pytest.mark.parametrize("T,N,K,f32", [(1, 3000, 4096, True), (4, 1000, 4096, True), (9, 1000, 5000, False), (60, 900, 4000, False), (300, 700, 4001, False),
                                       (1500, 2100, 2500, False), (100, 500, 9000, True)])
def test_steps(T, N, K, f32):
    """The sum's rounding and that of the scales' product are half a step of numbers that may be as large as the result's next
    power of two: a step of the result each at most, and half a step for the result's own. In all 3 2^-24, relatively."""
    note(f"steps {T} x {N} x {K}")
    rng = np.random.default_rng(K + T)
    i8 = vx.Int8Gemm(0)
    x, w = (rng.integers(60, 128, (n, K)).astype(np.int8) for n in (T, N))
    x[:, 0] = 127
    x[::3], w[1::2] = -x[::3], -w[1::2]
    sx, sw = (2.0 ** rng.uniform(-3, 3, n) for n in (T, N))
    sx, sw = sx.astype(np.float32), sw.astype(np.float32)
    out = torch.empty(T, N, device=DEV)
    if f32:  # (powers of two: the rows are quantized to these codes and scales)
        sx = np.float32(2.0) ** np.round(np.log2(sx)).astype(np.float32)
        xf = torch.tensor(x.astype(np.float32) * sx[:, None], device=DEV)
        i8.dispatch(out, xf, _rows(w, sw), workspace=i8.workspace(T, K))
    else:
        i8.dispatch(out, _rows(x, sx), _rows(w, sw))
    s = (torch.tensor(x, device=DEV).double() @ torch.tensor(w, device=DEV).double().t()).cpu().numpy()
    assert (np.abs(s) > 2 ** 24).mean() > 0.1
    ref = s * sx.astype(np.float64)[:, None] * sw.astype(np.float64)
    off = np.abs(out.cpu().numpy().astype(np.float64) - ref)
    assert (off <= np.abs(ref) * 3 * 2.0 ** -24 * (1 + 2.0 ** -22)).all(), (off / np.abs(ref)).max() * 2 ** 24
    steps = off / 2.0 ** (np.floor(np.log2(np.abs(ref))) - 23)
    assert steps.max() <= 2.5 * (1 + 2.0 ** -20), steps.max()
    note(f"{steps.max():.3f} steps, {(off / np.abs(ref)).max() * 2 ** 24:.3f} half steps relatively")
