"""Sizes that no launch has threads for are refused before any device work (CPU)."""
from __future__ import annotations

import ctypes as C

import pytest


@pytest.mark.parametrize("M, N", [((1 << 31) - 1, 1), (1 << 30, 300), (1 << 28, 5000)])
def test_products_of_more_tiles_than_a_launch_has_blocks(vs, M, N):
    """Tiles of 256 threads and 128 x 128 values at the largest, FP32."""
    lib, need = vs.load_library(), C.c_size_t(0)
    a = vs._LinearArgs(M=M, N=N, K=4, x=4096, w=4096, y=8192)
    assert lib.vcsr_linear(C.byref(a), None, None) == vs.VCSR_ERANGE
    assert lib.vcsr_linear_workspace(C.byref(a), C.byref(need)) == vs.VCSR_ERANGE
    g = vs._LinearGradArgs(M=M, N=4, K=N, dy=4096, x=8192, w=4096, dx=65536)
    assert lib.vcsr_linear_grad(C.byref(g), None, None) == vs.VCSR_ERANGE
    g.dw = 131072
    assert lib.vcsr_linear_grad_workspace(C.byref(g), C.byref(need)) == vs.VCSR_ERANGE


def test_products_of_just_fewer_pass_the_checks(vs):
    """2^30 rows of one tile: 64 x 64 tiles would be too many, larger ones are not."""
    lib, need = vs.load_library(), C.c_size_t(0)
    for M, N in ((1 << 30, 64), ((1 << 31) - 200, 1), (4, (1 << 31) - 300)):
        a = vs._LinearArgs(M=M, N=N, K=4, x=4096, w=4096, y=8192)
        assert lib.vcsr_linear_workspace(C.byref(a), C.byref(need)) == vs.VCSR_OK, (M, N)
        assert need.value == 0


def test_adamw_of_more_chunks_than_a_launch_has_blocks(vs):
    """2^24 chunks of 2,048 values, 256 threads each: in one tensor, and in two."""
    lib = vs.load_library()
    for sizes in ([1 << 35], [1 << 34, (1 << 34) - 2047]):
        t = (vs._AdamwTensor * len(sizes))(*[
            vs._AdamwTensor(n, 0, 0, 4096, 4096, 4096, 4096, None, None, None, 0.0) for n in sizes])
        out = C.c_void_p()
        assert lib.vcsr_adamw_create(t, len(sizes), None, C.byref(out)) == vs.VCSR_ERANGE, sizes
        assert not out.value
