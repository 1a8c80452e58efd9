"""Products of 8-bit integers with scales, plain and gated, against numpy: whole
numbers in 64 bits, codes by the definition's f32 operations."""
import math

import numpy as np
import pytest
import torch

import vortx_amd as vx
from tests.helpers import note

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
STEP = 2.0 ** -24  # half a step of f32, relative


@pytest.fixture(scope="module")
def i8():
    assert torch.cuda.is_available()
    return vx.Int8Gemm(0)


def _gpu(a):
    return torch.tensor(np.ascontiguousarray(a), device=DEV)


def _codes(x):
    """vx_i8_quantize in numpy, an f32 rounding for each operation."""
    x = x.astype(np.float32)
    m = np.abs(x).max(1, keepdims=True) if x.shape[1] else np.zeros((x.shape[0], 1), np.float32)
    with np.errstate(all="ignore"):
        small, bad = m < np.float32(2.0 ** -100), ~np.isfinite(m)
        r = np.where(small | bad, np.float32(0), np.float32(127) / m).astype(np.float32)
        d = np.where(bad, np.float32(np.nan), np.where(small, np.float32(0), (m / np.float32(127)).astype(np.float32)))
        q = np.where(bad, 0, np.clip(np.rint((x * r).astype(np.float32)), -127, 127))
    return q.astype(np.int8), d[:, 0].astype(np.float32), bad[:, 0]


def _rows(q, d, slack=0):
    """Int8Rows of these, with bytes of another value past the columns and between the rows."""
    rows, cols = q.shape
    stride = -(-max(cols, 1) // 16) * 16 + 16 * slack
    data = torch.full((max(rows, 1), stride), 113, dtype=torch.int8, device=DEV)[:rows]
    data[:, :cols] = _gpu(q)
    return vx.Int8Rows(data, _gpu(d), cols)


def _random(rng, T, N, K):
    x, w = rng.integers(-128, 128, (T, K)).astype(np.int8), rng.integers(-128, 128, (N, K)).astype(np.int8)
    return x, w, rng.uniform(0.001, 0.1, T).astype(np.float32), rng.uniform(0.001, 0.1, N).astype(np.float32)


def _exact(x, w, sx, sw):
    s = (torch.tensor(x).to(DEV).double() @ torch.tensor(w).to(DEV).double().t()).cpu().numpy()  # (whole numbers below 2^53)
    return s * sx.astype(np.float64)[:, None] * sw.astype(np.float64)


def _check(out, ref):
    """Three roundings of half a step each."""
    got = out.cpu().numpy().astype(np.float64)
    off = np.abs(got - ref) - np.abs(ref) * 3.01 * STEP
    assert np.isfinite(got).all() and (off <= 0).all(), (float(off.max()), np.argwhere(off > 0)[:5])


SIZES = [
    (1, 1, 1), (1, 16, 64), (1, 17, 15), (2, 100, 16), (1, 4096, 4096), (2, 333, 1000), (3, 65, 17), (5, 1, 300), (16, 40, 63), (16, 512, 2048),
    (17, 33, 65), (32, 100, 130), (31, 500, 777), (33, 70, 127), (64, 129, 512), (100, 300, 1100), (128, 64, 96), (127, 31, 4099),
    (129, 100, 64), (130, 257, 1), (200, 128, 63), (256, 300, 65), (300, 1000, 191), (257, 129, 16), (129, 1, 2000), (600, 513, 257),
    (1000, 2100, 130), (2049, 4200, 64), (1300, 8300, 200), (4097, 2500, 33),
]


@pytest.mark.parametrize("T,N,K", SIZES)
def test_product(i8, T, N, K):
    note(f"product {T} x {N} x {K}")
    rng = np.random.default_rng(T * 100 + N + K)
    x, w, sx, sw = _random(rng, T, N, K)
    ref = _exact(x, w, sx, sw)
    out = torch.full((T, N), float("nan"), device=DEV)
    i8.dispatch(out, _rows(x, sx), _rows(w, sw))
    _check(out, ref)
    # the same into a transposed view and a part of a wider one, from rows with room between them
    wide = torch.full((T + 2, N + 5), 7.5, device=DEV)
    i8.dispatch(wide[1:-1, 3:-2], _rows(x, sx, 1), _rows(w, sw, 3))
    assert torch.equal(wide[1:-1, 3:-2], out)
    wide[1:-1, 3:-2] = 7.5
    assert (wide == 7.5).all()
    turned = torch.empty(N, T, device=DEV).t()
    i8.dispatch(turned, _rows(x, sx), _rows(w, sw, 1))
    assert torch.equal(turned, out)


@pytest.mark.parametrize("T,N,K", [(1, 64, 131071), (20, 50, 131071), (140, 130, 131071)])
def test_the_longest_rows(i8, T, N, K):
    """All at -128: the largest sum there is, 131071 * 2^14, is still an int32."""
    x, w = np.full((T, K), -128, np.int8), np.full((N, K), -128, np.int8)
    w[0] = 127
    one = lambda n: np.ones(n, np.float32)  # noqa: E731
    out = torch.empty(T, N, device=DEV)
    i8.dispatch(out, _rows(x, one(T)), _rows(w, one(N)))
    _check(out, _exact(x, w, one(T), one(N)))


def _f32_case(rng, T, K):
    x = rng.standard_normal((T, K)).astype(np.float32)
    x[:, ::7] *= 8
    return x


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 4), (3, 7), (5, 1023), (4, 1024), (7, 4096), (2, 4099), (3, 5000), (2, 16384), (2, 16390), (520, 16390), (600, 4097),
                                       (1, 40003), (700, 130), (0, 5), (3, 0)])
def test_quantize(i8, rows, cols):
    note(f"quantize {rows} x {cols}")
    rng = np.random.default_rng(rows + cols)
    x = _f32_case(rng, rows, cols)
    x *= 10.0 ** rng.uniform(-20, 20, (rows, 1)).astype(np.float32)
    if rows > 2 and cols > 6:
        x[0] = 0
        x[1, :] = 1e-35
        x[2, 5] = 0.0
        x[2, :4] = [127, 2.5, 0.5, -1.5]  # ties
        x[2, 4:] = 0
    q, d, _ = _codes(x)
    for stride in (cols, cols + 3):  # rows 16-byte aligned, and not
        buf = torch.full((rows, max(stride, 1)), 9.0, device=DEV)
        buf[:, :cols] = _gpu(x)
        got = _rows(np.zeros((rows, cols), np.int8), np.zeros(rows, np.float32), 1)
        i8.quantize(got, buf[:, :cols])
        assert np.array_equal(got.data[:, :cols].cpu().numpy(), q) and np.array_equal(got.scales.cpu().numpy(), d)
        assert (got.data[:, cols:] == 113).all()
    if rows > 1 and cols > 1:
        i8.quantize(got, _gpu(x).t().contiguous().t())
        assert np.array_equal(got.data[:, :cols].cpu().numpy(), q) and np.array_equal(got.scales.cpu().numpy(), d)


@pytest.mark.parametrize("T,N,K", [(1, 100, 1), (1, 33, 63), (1, 512, 4096), (1, 70, 32768), (1, 70, 32769), (2, 40, 1000), (2, 48, 16384),
                                   (2, 48, 16385), (3, 40, 1000), (3, 1030, 129), (4, 700, 4096), (4, 50, 4097), (4, 300, 2049), (2, 90, 8192), (2, 5000, 8100), (3, 4300, 3333), (1, 70, 65536), (5, 40, 64), (1, 4200, 127), (16, 128, 4090), (40, 100, 515), (150, 200, 300), (513, 700, 129), (1, 16, 8191)])
def test_f32_rows_are_quantized_as_by_themselves(i8, T, N, K):
    """Bit for bit the product of vx_i8_quantize's rows, also from rows that are not aligned or not contiguous."""
    note(f"f32 rows {T} x {N} x {K}")
    rng = np.random.default_rng(T + N + K)
    x, (_, w, _, sw) = _f32_case(rng, T, K), _random(rng, 1, N, K)
    w = _rows(w, sw)
    q, d, _ = _codes(x)
    want, out = torch.empty(T, N, device=DEV), torch.empty(T, N, device=DEV)
    i8.dispatch(want, _rows(q, d), w)
    ws = i8.workspace(T, K)
    ws.fill_(255)
    gx = _gpu(x)
    odd = torch.full((T, K + 3), float("nan"), device=DEV)
    odd[:, 1:K + 1] = gx
    for view in (gx, odd[:, 1:K + 1], gx.t().contiguous().t(), (gx, vx.TensorLayout((T, K), (K, 1), 2, 0))):
        out.fill_(float("nan"))
        i8.dispatch(out, view, w, workspace=ws)
        assert torch.equal(out, want)


ACTS = {
    # value, and the bound of its relative error in half steps for a gate value g that is itself 3 of them off:
    # see the comments; y of the tanh form is 5 roundings and g's own 3 (times at most 3, the cube's) off
    "silu": (lambda g: g / (1 + np.exp(-g)), lambda g: 6 + 3 * (1 + np.abs(g))),
    "gelu_tanh": (lambda g: g / (1 + np.exp(-math.sqrt(8 / math.pi) * (g + 0.044715 * g ** 3))),
                  lambda g: 9 + 14 * np.abs(math.sqrt(8 / math.pi) * (g + 0.044715 * g ** 3))),
    # erfc: 16 steps allowed to the library's function; its argument, 4 half steps off, counts 2 z^2 + 2 = g^2 + 2 times
    "gelu": (lambda g: 0.5 * g * _erfc(-g / math.sqrt(2)), lambda g: 32 + 3 + 4 * (g * g + 2)),
    "relu": (lambda g: np.maximum(g, 0), lambda g: 3 + 0 * g),
}


def _erfc(z):
    return torch.erfc(torch.tensor(z, dtype=torch.float64)).numpy()


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("T,N,K", [(1, 1, 1), (1, 100, 300), (2, 17, 130), (9, 33, 65), (16, 200, 1000), (30, 31, 127), (77, 130, 64), (128, 40, 999),
                                   (129, 65, 130), (300, 100, 63), (257, 2100, 257), (2049, 2100, 70)])
def test_gated(i8, act, T, N, K):
    """sigmoid: e^-g to 3 half steps (the instruction's step and a rounding), 1 + e^-g one more, the reciprocal two; g's own 3
    count 1 + |g| times in g sigmoid(g); then u's 3 and two products. Below f32's normal numbers, 2^-125 of |g u|."""
    note(f"gated {act} {T} x {N} x {K}")
    rng = np.random.default_rng(T * 3 + N + K)
    x, w, sx, sw = _random(rng, T, 2 * N, K)
    sx, sw = sx * np.float32(20 / np.sqrt(K) / 73 ** 2 * 400), sw * np.float32(1)  # gates of a few units
    g, u = np.split(_exact(x, w, sx, sw), 2, axis=1)
    f, bound = ACTS[act]
    with np.errstate(over="ignore"):
        ref = f(g) * u
        tol = np.abs(ref) * (bound(g) + 5.1) * STEP + 2.0 ** -125 * (1 + np.abs(g * u))
    gate, up = _rows(w[:N], sw[:N]), _rows(w[N:], sw[N:], 2)
    out = torch.full((T, N), float("nan"), device=DEV)
    i8.dispatch_gated(out, _rows(x, sx), gate, up, act)
    off = np.abs(out.cpu().numpy().astype(np.float64) - ref) - tol
    assert (off <= 0).all(), (float(off.max()), np.argwhere(~(off <= 0))[:5], np.abs(g).max())
    wide = torch.full((T, N + 3), 7.5, device=DEV)
    i8.dispatch_gated(wide[:, 1:-2], _rows(x, sx, 1), gate, up, act)
    assert torch.equal(wide[:, 1:-2], out) and (wide[:, 0] == 7.5).all() and (wide[:, -2:] == 7.5).all()
    # from f32 rows: x as its rows stand for
    xf = _f32_case(rng, T, K)
    q, d, _ = _codes(xf)
    i8.dispatch_gated(out, _rows(q, d), gate, up, act)
    again = torch.empty(T, N, device=DEV)
    i8.dispatch_gated(again, _gpu(xf), gate, up, act, workspace=i8.workspace(T, K))
    assert torch.equal(out, again)


@pytest.mark.parametrize("T", [1, 2, 20, 60, 150, 1200])
def test_what_is_not_finite_stays_in_its_row_and_column(i8, T):
    rng = np.random.default_rng(T)
    N, K = 2100, 200
    xf, wf = _f32_case(rng, T, K), _f32_case(rng, N, K)
    clean = torch.empty(T, N, device=DEV)
    w = vx.Int8Rows.empty(N, K)
    ws = i8.workspace(T, K)
    i8.quantize(w, _gpu(wf))
    i8.dispatch(clean, _gpu(xf), w, workspace=ws)
    bad_x, bad_w = xf.copy(), wf.copy()
    bad_x[T // 2, 3], bad_w[77, 5], bad_w[1999, 199] = np.inf, np.nan, -np.inf
    i8.quantize(w, _gpu(bad_w))
    out = torch.empty(T, N, device=DEV)
    i8.dispatch(out, _gpu(bad_x), w, workspace=ws)
    keep_t, keep_n = torch.arange(T, device=DEV) != T // 2, torch.ones(N, dtype=torch.bool, device=DEV)
    keep_n[[77, 1999]] = False
    assert out[T // 2].isnan().all() and out[:, ~keep_n].isnan().all()
    assert torch.equal(out[keep_t][:, keep_n], clean[keep_t][:, keep_n])


@pytest.mark.parametrize("T", [1, 9, 40, 200])
def test_scales_far_from_one(i8, T):
    """Where a product of two of three factors leaves f32's range, the result is still the rounded one."""
    rng = np.random.default_rng(T)
    N, K = 64, 128
    x, w, sx, sw = _random(rng, T, N, K)
    w[3] = 0
    big, small = np.float32(1e36), np.float32(1e-36)
    for a, b in ((big, small), (small, big), (big, np.float32(1e-40)), (small, np.float32(1e-3)), (big, np.float32(1.0))):
        out = torch.empty(T, N, device=DEV)
        i8.dispatch(out, _rows(x, sx * a), _rows(w, sw * b))
        ref = _exact(x, w, (sx * a).astype(np.float32), (sw * b).astype(np.float32))
        with np.errstate(over="ignore"):
            ref32 = ref.astype(np.float32)
        got = out.cpu().numpy()
        ok = (got == ref32) | (np.abs(got.astype(np.float64) - ref) <= np.abs(ref) * 3.01 * STEP + 2.0 ** -149)
        assert ok.all() and (got[:, 3] == 0).all()


def test_two_streams_and_a_graph(i8):
    rng = np.random.default_rng(0)
    T, N, K = 40, 700, 900
    x, (_, w, _, sw) = _f32_case(rng, T, K), _random(rng, 1, N, K)
    w = _rows(w, sw)
    want, out = torch.empty(T, N, device=DEV), [torch.empty(T, N, device=DEV) for _ in range(2)]
    gx, ws = _gpu(x), [i8.workspace(T, K) for _ in range(2)]
    i8.dispatch(want, gx, w, workspace=ws[0])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, o, b in zip(streams, out, ws):
            with torch.cuda.stream(s):
                i8.dispatch(o, gx, w, workspace=b)
    torch.cuda.synchronize()
    assert torch.equal(out[0], want) and torch.equal(out[1], want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        i8.dispatch(out[0], gx, w, workspace=ws[0])
    for seed in range(3):
        gx.copy_(_gpu(_f32_case(np.random.default_rng(seed + 5), T, K)))
        i8.dispatch(want, gx, w, workspace=ws[1])
        out[0].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want)


def test_empty_and_refused(i8):
    w, x = vx.Int8Rows.empty(32, 64), torch.zeros(6, 64, device=DEV)  # (more tokens than go without a workspace)
    up = vx.Int8Rows.empty(32, 64)
    ws = i8.workspace(6, 64)
    assert [i8.workspace_size(*n) > 0 for n in ((4, 4096), (2, 8192), (1, 65536), (5, 128), (4, 4097), (2, 8193), (1, 65537))] == [False] * 3 + [True] * 4
    i8.dispatch(torch.empty(0, 32, device=DEV), torch.empty(0, 64, device=DEV), w)
    i8.dispatch(torch.empty(6, 0, device=DEV), x, vx.Int8Rows.empty(0, 64), workspace=ws)
    out = torch.empty(6, 32, device=DEV)
    for call in [lambda: i8.dispatch(out, x, w),                                            # no workspace
                 lambda: i8.dispatch(out, x, w, workspace=ws[:16]),
                 lambda: i8.dispatch(out, x, w, workspace=torch.empty(4096, dtype=torch.uint8, device=DEV)[1:]),
                 lambda: i8.dispatch(out, x[:, :60], w, workspace=ws),
                 lambda: i8.dispatch(out[:, :31], x, w, workspace=ws),
                 lambda: i8.dispatch(out[:3], x, w, workspace=ws),
                 lambda: i8.dispatch(out[:1].expand(6, 32), x, w, workspace=ws),
                 lambda: i8.dispatch(out[None].expand(2, 6, 32), x, w, workspace=ws),
                 lambda: i8.dispatch_gated(out, x, w, up, "tanh", workspace=ws),
                 lambda: i8.dispatch_gated(out, x, w, vx.Int8Rows.empty(33, 64), workspace=ws),
                 lambda: i8.dispatch_gated(out, x, w, vx.Int8Rows.empty(32, 65), workspace=ws),
                 lambda: i8.dispatch(out, torch.zeros(6, 0, device=DEV), vx.Int8Rows.empty(32, 0), workspace=ws),
                 lambda: i8.dispatch(out, vx.Int8Rows.empty(6, 131072), vx.Int8Rows.empty(32, 131072)),
                 lambda: i8.quantize(w, x),
                 lambda: vx.Int8Rows(torch.zeros(4, 24, dtype=torch.int8, device=DEV), torch.zeros(3, device=DEV)),
                 lambda: vx.Int8Rows(torch.zeros(2, 20, dtype=torch.int8, device=DEV), torch.zeros(2, device=DEV)),   # the last row ends too early
                 lambda: vx.Int8Rows(torch.zeros(32, 4, dtype=torch.int8, device=DEV).t(), torch.zeros(4, device=DEV)),
                 lambda: vx.Int8Rows(torch.zeros(4, 32, dtype=torch.int8, device=DEV), torch.zeros(4, device=DEV), 33)]:
        with pytest.raises(vx.VortxError):
            call()
    odd = vx.Int8Rows(torch.zeros(6, 24, dtype=torch.int8, device=DEV), torch.zeros(6, device=DEV), 8)
    with pytest.raises(vx.VortxError):
        i8.quantize(odd, x[:, :8])
    for call in [lambda: i8.dispatch(out, x.double(), w, workspace=ws), lambda: i8.dispatch(out.half(), x, w, workspace=ws),
                 lambda: i8.dispatch(out, x, w, workspace=torch.empty(4096, dtype=torch.uint8)), lambda: i8.dispatch_gated(out, x, w, None),
                 lambda: vx.Int8Rows(torch.zeros(4, 32, device=DEV), torch.zeros(4, device=DEV)),
                 lambda: vx.Int8Rows(torch.zeros(4, 32, dtype=torch.int8, device=DEV), torch.zeros(4, device=DEV).double())]:
        with pytest.raises(TypeError):
            call()


@pytest.mark.parametrize("T", [1, 4, 20, 60, 150])
@pytest.mark.parametrize("rows,stride", [(70000, 65536), (300, 1 << 24)])
def test_weights_past_32_bits(i8, T, rows, stride):
    """Rows of 192 columns whose places pass 2^32 bytes."""
    note(f"far weights {T} by {rows} rows {stride} bytes apart")
    rng = np.random.default_rng(T)
    K, n = 192, 300
    data = torch.empty(rows, stride, dtype=torch.int8, device=DEV)
    x, w, sx, sw = _random(rng, T, n, K)
    data[-n:, :K] = _gpu(w)
    weights = vx.Int8Rows(data, torch.cat([torch.ones(rows - n, device=DEV), _gpu(sw)]), K)
    out = torch.empty(T, rows, device=DEV)
    i8.dispatch(out, _rows(x, sx), weights)
    _check(out[:, -n:], _exact(x, w, sx, sw))
    xf = _gpu(_f32_case(rng, T, K))
    q = vx.Int8Rows.empty(T, K)
    i8.quantize(q, xf)
    i8.dispatch(out, xf, weights, workspace=i8.workspace(T, K))
    _check(out[:, -n:], _exact(q.data[:, :K].cpu().numpy(), w, q.scales.cpu().numpy(), sw))


def test_tokens_past_32_bits(i8):
    rng = np.random.default_rng(8)
    T, N, K, stride = 300, 50, 200, 1 << 24
    data = torch.empty(T, stride, dtype=torch.int8, device=DEV)
    x, w, sx, sw = _random(rng, T, N, K)
    data[:, :K] = _gpu(x)
    out = torch.empty(T, N, device=DEV)
    i8.dispatch(out, vx.Int8Rows(data, _gpu(sx), K), _rows(w, sw))
    _check(out, _exact(x, w, sx, sw))
    i8.quantize(vx.Int8Rows(data, torch.empty(T, device=DEV), K), _gpu(x * sx[:, None]))
    want, _, _ = _codes(x * sx[:, None])
    assert np.array_equal(data[:, :K].cpu().numpy(), want)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("T,N,K", [(17, 200, 1030), (100, 4096, 11008), (33, 65, 5000), (128, 1000, 4096), (129, 129, 2049), (300, 500, 8191),
                                   (1000, 130, 16385), (64, 3, 131071), (70, 4097, 1100), (1024, 256, 2048), (20, 31, 1024), (2000, 200, 4100),
                                   (5000, 100, 1500)])
def test_parts_of_long_rows(i8, T, N, K, gated):
    """Sums of parts of K, joined: the bits of the product of vx_i8_quantize's rows, with any contents of the workspace."""
    note(f"parts {T} x {N} x {K} gated {gated}")
    rng = np.random.default_rng(T + N + K)
    x = _gpu(_f32_case(rng, T, K))
    x[T // 2, K - 1] = float("nan")
    w, up = (vx.Int8Rows.empty(N, K) for _ in range(2))
    for r in (w, up):
        r.data.copy_(torch.randint(-128, 128, r.data.shape, dtype=torch.int8, device=DEV))
        r.scales.copy_(torch.rand(N, device=DEV) + 0.01)
    q = vx.Int8Rows.empty(T, K)
    q.data.fill_(77)
    i8.quantize(q, x)
    ws = i8.workspace(T, K)
    want, got = torch.empty(T, N, device=DEV), torch.full((N, T + 1), 7.0, device=DEV)
    call = (lambda o, r, **k: i8.dispatch_gated(o, r, w, up, "silu", **k)) if gated else (lambda o, r, **k: i8.dispatch(o, r, w, **k))
    call(want, q)
    for fill, out in ((255, torch.empty(T, N, device=DEV)), (0, got.t()[:T])):
        ws.fill_(fill)
        call(out, x, workspace=ws)
        assert torch.equal(out.nan_to_num(3.0), want.nan_to_num(3.0))
    assert (got[:, T] == 7.0).all() and want[T // 2].isnan().all() and not want[0].isnan().any()
    if T <= 1000:  # (a workspace for more tokens and columns)
        out = torch.empty(T, N, device=DEV)
        call(out, x, workspace=i8.workspace(T + 1100, K + 50))
        assert torch.equal(out.nan_to_num(3.0), want.nan_to_num(3.0))
    if not gated:
        _check(want[:2], _exact(q.data[:2, :K].cpu().numpy(), w.data[:, :K].cpu().numpy(), q.scales[:2].cpu().numpy(), w.scales.cpu().numpy()))
