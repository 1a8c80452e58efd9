"""Products of 8-bit integers with a scale for each token and channel.

:class:`Int8Rows` holds rows of integers with an f32 scale each, activations
(a scale a token) as well as weights (a scale a channel); :class:`Int8Gemm` makes
them of f32 rows and multiplies them on the int8 matrix cores, with exact sums,
plain or as the gated half of a feed-forward block (``vx_i8_quantize`` and
what follows it in include/vortx_hip.h; the reference has none of this)::

    gate, up, down = (vx.Int8Rows.empty(*w.shape) for w in (wg, wu, wd))
    i8 = vx.Int8Gemm(0)
    i8.quantize(gate, wg)                         # once: f32 [channels, cols]
    ...
    ws = i8.workspace(tokens, max(hidden, inner))
    i8.dispatch_gated(h, x, gate, up, act="silu", workspace=ws)  # x [tokens, hidden], h [tokens, inner]
    i8.dispatch(y, h, down, workspace=ws)
"""
from __future__ import annotations

import ctypes as C

import vortx_amd as _vx

from . import _ADDR, _ByAddress, _Context, _ffi, _stream, _view_of
from ._ffi import VortxError, check, lib

_QUANTIZE, _ROWS, _X, _GATED, _GATED_X = (_ADDR[n] for n in ("vx_i8_quantize", "vx_gemm_i8", "vx_gemm_i8_x", "vx_gemm_i8_gated",
                                                             "vx_gemm_i8_gated_x"))
_ACTS = {"silu": 0, "gelu_tanh": 1, "gelu": 2, "relu": 3}


class Int8Rows(_ByAddress):
    """``rows`` x ``cols`` integers, ``data`` (int8 GPU tensor [rows, at least
    cols], neighbours in a row next to each other, rows a multiple of 16 bytes
    apart and 16-byte aligned), with ``scales`` (f32 [rows]) for the values
    scales * data. A row's last 16 bytes have to lie in the tensor whole."""

    def __init__(self, data, scales, cols: int | None = None):
        import torch
        if not (isinstance(data, torch.Tensor) and data.is_cuda and data.dtype == torch.int8 and data.dim() == 2):
            raise TypeError("data must be an int8 tensor [rows, cols] on the GPU")
        if not (isinstance(scales, torch.Tensor) and scales.is_cuda and scales.dtype == torch.float32):
            raise TypeError("scales must be a float32 tensor on the GPU")
        rows = data.shape[0]
        cols = data.shape[1] if cols is None else cols
        if not 0 <= cols <= data.shape[1]:
            raise VortxError(_ffi.VX_ERR_SHAPE, f"{cols} columns of rows of {data.shape[1]}")
        if scales.shape != (rows,) or not scales.is_contiguous():
            raise VortxError(_ffi.VX_ERR_SHAPE, f"scales is {tuple(scales.shape)}, not one row of {rows}")
        if data.shape[1] > 1 and data.stride(1) != 1:
            raise VortxError(_ffi.VX_ERR_UNSUPPORTED, "data has strided elements")
        stride = data.stride(0) if rows > 1 else -(-max(cols, 1) // 16) * 16
        if stride < cols:
            raise VortxError(_ffi.VX_ERR_UNSUPPORTED, "data has overlapping rows")
        room = data.untyped_storage().nbytes() - data.storage_offset()
        need = (rows - 1) * stride + -(-cols // 16) * 16
        if rows and cols and room < need:
            raise VortxError(_ffi.VX_ERR_INVALID, f"rows of 16 bytes' multiples need {need} bytes, the buffer holds {room}")
        self.data, self.scales, self.rows, self.cols = data, scales, rows, cols
        self._c = _ffi.VxI8Rows(data.data_ptr() or None, scales.data_ptr() or None, stride, rows, cols)
        self._at = C.addressof(self._c)

    @staticmethod
    def empty(rows: int, cols: int, device="cuda:0") -> "Int8Rows":
        """New ones of undefined contents, rows a multiple of 128 bytes apart."""
        import torch
        data = torch.empty(rows, -(-max(cols, 1) // 128) * 128, dtype=torch.int8, device=device)
        return Int8Rows(data, torch.empty(rows, dtype=torch.float32, device=device), cols)

    def values(self):
        """What they stand for, f32 [rows, cols]."""
        return self.data[:, :self.cols].float() * self.scales[:, None]


def _rows(name, v):
    """Calls take an Int8Rows by its address: nothing else has one that they could read."""
    if not isinstance(v, Int8Rows):
        raise TypeError(f"{name} must be Int8Rows")


class Int8Gemm(_Context):
    """Products of :class:`Int8Rows`."""

    def quantize(self, out: Int8Rows, x, stream=None) -> None:
        """The rows of ``x`` (f32 [rows, cols] view) as integers with a scale
        each, max|x| / 127 (vx_i8_quantize)."""
        _rows("out", out)
        st = _vx._pycall.i8_quantize(_QUANTIZE, self._ctx, stream, out._at, x)
        if st is not None:
            if st:
                check(st)
            return
        xv = _view_of(x, False)
        check(lib().vx_i8_quantize(self._h, _stream(stream), C.byref(out._c), C.byref(xv)))

    @staticmethod
    def workspace_size(tokens: int, cols: int) -> int:
        """Bytes of workspace for ``tokens`` f32 rows of ``cols`` values (0: none)."""
        for n in (tokens, cols):
            if not 0 <= n < 2 ** 32:
                raise VortxError(_ffi.VX_ERR_INVALID, f"{n}: a number from 0 to 2^32 - 1 is expected")
        n = C.c_uint64()
        check(lib().vx_gemm_i8_ws_size(tokens, cols, C.byref(n)))
        return n.value

    @staticmethod
    def workspace(tokens: int, cols: int, device="cuda:0"):
        """A workspace for :meth:`dispatch` and :meth:`dispatch_gated` of f32
        rows: enough for up to so many tokens and columns."""
        import torch
        return torch.empty(max(16, Int8Gemm.workspace_size(tokens, cols)), dtype=torch.uint8, device=device)

    def dispatch(self, out, x, w: Int8Rows, workspace=None, stream=None) -> None:
        """``out`` [T, N] = ``x`` [T, K] times the transpose of ``w`` [N, K].
        ``x``: :class:`Int8Rows`, or an f32 view, whose rows are quantized first
        (for one to four tokens within the product, else into ``workspace``,
        which is for f32 views alone: rows that are integers need none)."""
        self._run(out, x, w, None, 0, workspace, stream)

    def dispatch_gated(self, out, x, gate: Int8Rows, up: Int8Rows, act: str = "silu", workspace=None, stream=None) -> None:
        """``out`` = act(x gate^T) * (x up^T), ``act`` one of "silu",
        "gelu_tanh", "gelu", "relu"; ``x`` as in :meth:`dispatch`."""
        if act not in _ACTS:
            raise VortxError(_ffi.VX_ERR_INVALID, f"act is {act!r}: one of {', '.join(_ACTS)} is expected")
        _rows("up", up)
        self._run(out, x, gate, up, _ACTS[act], workspace, stream)

    def _run(self, out, x, w, up, act, workspace, stream):
        _rows("weights", w)
        rows = isinstance(x, Int8Rows)
        fn = (_ROWS if rows else _X) if up is None else (_GATED if rows else _GATED_X)
        st = _vx._pycall.gemm_i8(fn, self._ctx, stream, out, x._at if rows else None, x, w._at, None if up is None else up._at, act,
                                 workspace)
        if st is not None:
            if st:
                check(st)
            return
        ov = _view_of(out, True)
        weights = (C.byref(w._c),) if up is None else (C.byref(w._c), C.byref(up._c), act)
        if rows:
            f = lib().vx_gemm_i8 if up is None else lib().vx_gemm_i8_gated
            check(f(self._h, _stream(stream), C.byref(ov), C.byref(x._c), *weights))
            return
        import torch
        ws, nbytes = None, 0
        if workspace is not None:
            if not (isinstance(workspace, torch.Tensor) and workspace.is_cuda and workspace.is_contiguous()):
                raise TypeError("workspace must be a contiguous GPU tensor")
            ws, nbytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        xv = _view_of(x, False)
        f = lib().vx_gemm_i8_x if up is None else lib().vx_gemm_i8_gated_x
        check(f(self._h, _stream(stream), C.byref(ov), C.byref(xv), *weights, ws, nbytes))
