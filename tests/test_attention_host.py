"""Host side of the quantized cache and the attention over it, without a GPU."""
import ctypes as C

import pytest

import vortx_amd as vx
from vortx_amd import _ffi


@pytest.mark.parametrize("k,v,dim,per", [(vx.VX_Q8_0, vx.VX_Q8_0, 128, 272), (vx.VX_Q8_0, vx.VX_Q4_0, 64, 104),
                                         (vx.VX_Q4_0, vx.VX_Q4_0, 96, 108), (vx.VX_Q4_0, vx.VX_Q8_0, 256, 416)])
def test_cache_size(k, v, dim, per):
    assert vx.kv_cache_size(3, 32, 5, dim, k, v) == 3 * 32 * 5 * (per + 2)
    assert vx.kv_cache_size(0, 32, 5, dim, k, v) == 0


@pytest.mark.parametrize("change,status", [
    (dict(dim=80), _ffi.VX_ERR_UNSUPPORTED), (dict(dim=512), _ffi.VX_ERR_UNSUPPORTED),
    (dict(page_tokens=8), _ffi.VX_ERR_UNSUPPORTED), (dict(page_tokens=48), _ffi.VX_ERR_UNSUPPORTED),
    (dict(heads=0), _ffi.VX_ERR_UNSUPPORTED), (dict(k_type=vx.VX_Q4_K), _ffi.VX_ERR_INVALID),
    (dict(v_type=0), _ffi.VX_ERR_INVALID), (dict(pages=1 << 31, page_tokens=16), _ffi.VX_ERR_UNSUPPORTED)])
def test_cache_refusals(change, status):
    with pytest.raises(vx.VortxError) as e:
        vx.kv_cache_size(**{**dict(pages=2, page_tokens=16, heads=1, dim=64), **change})
    assert e.value.status == status


def test_null_arguments():
    lib, n = vx.lib(), C.c_uint64()
    assert lib.vx_kv_cache_size(None, C.byref(n)) == _ffi.VX_ERR_INVALID
    assert lib.vx_kv_write(None, None, None, None, None, None) == _ffi.VX_ERR_INVALID
    assert lib.vx_kv_read(None, None, None, None, None, None) == _ffi.VX_ERR_INVALID
    assert lib.vx_attention(None, None, None, None, None, None, None, None, 0) == _ffi.VX_ERR_INVALID
    assert lib.vx_attention_tree(None, None, None, None, None, None, None, None, 0, 0, None, 0) == _ffi.VX_ERR_INVALID
    assert lib.vx_attention_ws_size(None, None, None, None, 1, 1, C.byref(n)) == _ffi.VX_ERR_INVALID
