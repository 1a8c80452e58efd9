"""Where pages and steps keep their numbers, on the CPU."""
import pytest

import vortx_amd as vx


def test_pages_and_steps_are_on_the_gpu():
    """(resize hands their addresses to kernels)"""
    for make in (lambda: vx.KvPages(4, 16, 2, 2, device="cpu"), lambda: vx.KvStep(2, 3, device="cpu"), lambda: vx.KvPages(0, 16, 0, 0, device="cpu"),
                 lambda: vx.KvStep(0, 0, device="cpu"), lambda: vx.KvStep(2, 3, device="meta")):
        with pytest.raises(TypeError):
            make()
