"""What the fast calls of 8-bit products, and of caches, make of arguments of a wrong type, on the
CPU: tensors are stand-ins with a tensor's attributes, the C functions are counted."""
import subprocess
import sys

import pytest

import vortx_amd as vx
from tests.test_int8_host import ROOT

CHILD = """
import ctypes as C
import torch
import vortx_amd as vx
from vortx_amd import _ffi, attention, int8

class Tensor:  # 4 x 8 values "on the GPU"
    dtype, is_cuda, shape = torch.float32, True, (4, 8)
    def __init__(self, *shape):
        if shape: self.shape = shape
    def stride(self): return (16, 8, 1)[-len(self.shape):]
    def data_ptr(self): return 4096
    def is_contiguous(self): return True
    nbytes = 128
class Stream:
    cuda_stream = 0

vx._pycall.setup(vx.QWeight, Tensor, torch.float32, None, None, torch.int32)
calls = []
def stands_for(name, n):
    f = C.CFUNCTYPE(C.c_int, *[C.c_uint64] * n)(lambda *a: calls.append((name, a)) or 0)
    return f, C.cast(f, C.c_void_p).value
made = {n: stands_for(n, k) for n, k in (("_ROWS", 5), ("_X", 7), ("_GATED", 7), ("_GATED_X", 9), ("_QUANTIZE", 4))}
for n, (_, at) in made.items():
    setattr(int8, n, at)
i8 = int8.Int8Gemm.__new__(int8.Int8Gemm)
i8._ctx, i8._h = 8, C.c_void_p(8)

def rows():
    r = int8.Int8Rows.__new__(int8.Int8Rows)
    r._c = _ffi.VxI8Rows(4096, 4096, 16, 4, 8)
    r._at = C.addressof(r._c)
    return r

x, w, up, out, st = rows(), rows(), rows(), Tensor(), Stream()
def only(name):
    global calls
    got, calls = calls, []
    assert [c[0] for c in got] == [name], got
i8.dispatch(out, x, w, stream=st); only("_ROWS")
i8.dispatch(out, Tensor(), w, workspace=Tensor(), stream=st); only("_X")
i8.dispatch_gated(out, x, w, up, stream=st); only("_GATED")
i8.dispatch_gated(out, Tensor(), w, up, workspace=Tensor(), stream=st); only("_GATED_X")
i8.quantize(w, Tensor(), stream=st); only("_QUANTIZE")
keep = C.create_string_buffer(256)  # (a number that is an address is still no tensor)
cache = attention.KvCache.__new__(attention.KvCache)
cache._c = _ffi.VxKvCache(4096, 0, 0, 16, 1, 64, 1, 1)
cache._addr = C.addressof(cache._c)
for bad in (C.addressof(keep), 5, True, None, cache, "x", 1.5):
    for call in (lambda: i8.dispatch(out, bad, w, stream=st), lambda: i8.dispatch_gated(out, bad, w, up, stream=st),
                 lambda: i8.dispatch(out, x, bad, stream=st), lambda: i8.dispatch_gated(out, x, bad, up, stream=st),
                 lambda: i8.dispatch_gated(out, x, w, bad, stream=st), lambda: i8.quantize(bad, Tensor(), stream=st),
                 lambda: i8.dispatch(out, Tensor(), bad, workspace=Tensor(), stream=st)):
        try:
            call()
        except TypeError:
            pass
        else:
            raise AssertionError(f"{bad!r} is taken")
        assert not calls, (bad, calls)
# and what has the address of something else is no cache
for n, k in (("_WRITE", 7), ("_READ", 7), ("_WRITE_ROTATED", 9)):
    made[n] = stands_for(n, k)
    setattr(attention, n, made[n][1])
kv = attention.KvAttention.__new__(attention.KvAttention)
kv._ctx, kv._h = 8, C.c_void_p(8)
h, slots = Tensor(4, 2, 8), Tensor(4)
slots.dtype = torch.int32
slots.stride = lambda: (1,)
how = attention.Rotation(0, 0, 0, (), _ffi.VxRotation())
kv.write(cache, h, h, slots, stream=st); only("_WRITE")
kv.read(h, h, cache, slots, stream=st); only("_READ")
kv.write_rotated(cache, h, h, h, h, None, slots, how, stream=st); only("_WRITE_ROTATED")
pages = attention.KvPages.__new__(attention.KvPages)
pages._c = _ffi.VxKvPages(4096, 4096, 4096, 4096, 2, 2, 2, 16, 4, 0)
pages._at = C.addressof(pages._c)
for bad in (rows(), pages, how, st):
    for call in (lambda: kv.write(bad, h, h, slots, stream=st), lambda: kv.read(h, h, bad, slots, stream=st),
                 lambda: kv.write_rotated(bad, h, h, h, h, None, slots, how, stream=st)):
        try:
            call()
        except (TypeError, AttributeError):
            pass
        else:
            raise AssertionError(f"{bad!r} is taken")
        assert not calls, (bad, calls)
print("fine")
"""


def test_arguments_of_a_wrong_type():
    if not hasattr(vx._pycall, "__file__"):
        pytest.skip("without the C binding")
    r = subprocess.run([sys.executable, "-c", CHILD], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "fine" in r.stdout, (r.stdout + r.stderr)[-3000:]
