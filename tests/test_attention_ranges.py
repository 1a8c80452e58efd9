"""Numbers that do not fit the library's 32-bit fields are refused, not taken as others."""
import pytest
import torch

import vortx_amd as vx
from vortx_amd import _ffi


@pytest.mark.parametrize("change", [dict(pages=2 ** 32 + 2), dict(pages=-1), dict(page_tokens=2 ** 32 + 16), dict(heads=2 ** 32 + 1),
                                    dict(dim=2 ** 32 + 64), dict(k_type=2 ** 32 + vx.VX_Q8_0), dict(v_type=-2 ** 32 + vx.VX_Q8_0)])
def test_cache(change):
    with pytest.raises(vx.VortxError, match=next(iter(change))) as e:
        vx.kv_cache_size(**{**dict(pages=2, page_tokens=16, heads=1, dim=64), **change})
    assert e.value.status == _ffi.VX_ERR_INVALID


@pytest.mark.gpu
@pytest.mark.parametrize("change", [dict(window=-1), dict(window=2 ** 32 + 5), dict(max_len=2 ** 32 + 10), dict(max_len=-1),
                                    dict(max_queries=2 ** 32 + 1), dict(q_heads=2 ** 32 + 2), dict(tokens=2 ** 32)])
def test_plan(change):
    kv, dev = vx.KvAttention(0), torch.device("cuda:0")
    cache = vx.KvCache(4, 16, 2, 64)
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    args = (cache, i32([0, 1]), i32(20), i32(0, 1))
    fine = dict(q_heads=2, max_queries=1, max_len=32)
    kv.plan(*args, **fine)
    with pytest.raises(vx.VortxError, match=next(iter(change))) as e:
        kv.plan(*args, **{**fine, **change})
    assert e.value.status == _ffi.VX_ERR_INVALID
