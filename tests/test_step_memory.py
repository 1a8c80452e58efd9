"""Where pages and steps keep their numbers, on the CPU."""
import pytest

import vortx_amd as vx


def test_pages_and_steps_are_on_the_gpu():
    """(resize hands their addresses to kernels)"""
    for make in (lambda: vx.KvPages(4, 16, 2, 2, device="cpu"), lambda: vx.KvStep(2, 3, device="cpu"), lambda: vx.KvPages(0, 16, 0, 0, device="cpu"),
                 lambda: vx.KvStep(0, 0, device="cpu"), lambda: vx.KvStep(2, 3, device="meta")):
        with pytest.raises(TypeError):
            make()


def test_what_a_call_takes_by_address_is_not_replaced():
    """A tensor put in the place of another would leave calls with the address of memory that is free."""
    from vortx_amd import _ffi, attention, int8
    pages, step, rows = (c.__new__(c) for c in (vx.KvPages, vx.KvStep, int8.Int8Rows))
    for o, names in ((pages, "table lens free free_count pages seqs cols page_tokens _c"), (step, "starts slots positions tokens seqs"),
                     (rows, "data scales rows cols _c")):
        for n in names.split():
            setattr(o, n, 1)  # (as their own making does)
            for bad in (2, None):
                with pytest.raises(AttributeError, match=n):
                    setattr(o, n, bad)
            assert getattr(o, n) == 1
        o.label = "what else a program keeps there"
    how = attention.Rotation(0, 0, 0, (), _ffi.VxRotation())
    for n in ("dim", "q_heads", "k_heads", "keep", "_c", "_call"):
        with pytest.raises(AttributeError, match=n):
            setattr(how, n, getattr(how, n))
