"""Arguments the dense operators refuse, before any device work (CPU)."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest


class Fake:
    """A buffer that is described and never touched."""

    def __init__(self, shape, dtype=np.float32, ptr=4096, nbytes=None, ld=None):
        self.shape, self.dtype = tuple(np.atleast_1d(shape)), np.dtype(dtype)
        self.ptr = C.c_void_p(ptr)
        if ld is not None:
            self.ld = ld
        n = int(np.prod(self.shape)) if ld is None else (self.shape[0] - 1) * ld + self.shape[1]
        self.nbytes = n * self.dtype.itemsize if nbytes is None else nbytes


def mat(*shape, **kw):
    return Fake(shape, **kw)


def bf(*shape, **kw):
    return Fake(shape, np.uint16, **kw)


def f8(*shape, **kw):
    return Fake(shape, np.uint8, **kw)


def refused(vs, code, fn, *args, **kw):
    with pytest.raises(vs.VcsrError) as e:
        fn(*args, **kw)
    assert e.value.code == code, e.value


NORM = {
    "y of another shape": dict(y=mat(4, 7)),
    "x of no known type": dict(x=Fake((4, 8), np.int32)),
    "8-bit x": dict(x=f8(4, 8)),
    "residual of another type": dict(residual=bf(4, 8)),
    "sum of another type": dict(sum=bf(4, 8)),
    "short weight": dict(weight=mat(7)),
    "weight of bf16": dict(weight=bf(8)),
    "stride under the row": dict(x=mat(4, 8, ld=6, nbytes=4096)),
    "x too short for its stride": dict(x=mat(4, 8, ld=64, nbytes=128)),
    "negative eps": dict(eps=-1e-6),
    "eps not finite": dict(eps=float("nan")),
    "8-bit y without scales": dict(y=f8(4, 8)),
    "scales without 8-bit y": dict(y_scale=mat(4)),
    "short scales": dict(y=f8(4, 8), y_scale=mat(3)),
    "no x": dict(x=mat(4, 8, ptr=0)),
    "no y": dict(y=mat(4, 8, ptr=0)),
    "misaligned x": dict(x=mat(4, 8, ptr=4098)),
    "misaligned rstd": dict(rstd=mat(4, ptr=4097)),
    "y over x of another type": dict(x=mat(4, 8, ptr=8192), y=bf(4, 8, ptr=8192)),
    "y over residual of another type": dict(residual=mat(4, 8, ptr=8192), y=bf(4, 8, ptr=8192)),
    "sum over y": dict(sum=mat(4, 8, ptr=65536)),
    "sum over x of another stride": dict(x=mat(4, 8, ptr=8192),
                                         sum=mat(4, 8, ptr=8192, ld=9, nbytes=4096)),
    "no columns": dict(x=mat(4, 0), y=mat(4, 0), weight=mat(0)),
}


@pytest.mark.parametrize("case", NORM)
def test_rmsnorm_refuses(vs, case):
    kw = dict(x=mat(4, 8), weight=mat(8), y=mat(4, 8, ptr=65536))
    kw.update(NORM[case])
    refused(vs, vs.VCSR_EINVAL, vs.run_rmsnorm_gpu, **kw)


GRAD = {
    "dy of another shape": dict(dy=mat(4, 9)),
    "8-bit dy": dict(dy=f8(4, 8)),
    "dx of another type": dict(dx=bf(4, 8)),
    "no rstd": dict(rstd=None),
}


@pytest.mark.parametrize("case", GRAD)
def test_rmsnorm_grad_refuses(vs, case):
    kw = dict(dy=mat(4, 8), s=mat(4, 8), weight=mat(8), rstd=mat(4), dx=mat(4, 8))
    kw.update(GRAD[case])
    refused(vs, vs.VCSR_EINVAL, vs.run_rmsnorm_grad_gpu, **kw)


@pytest.mark.parametrize("ws", [f8(16), f8(1 << 20, ptr=4104)], ids=["short", "misaligned"])
def test_rmsnorm_grad_refuses_a_workspace(vs, ws):
    """Many rows: dweight goes through partial sums."""
    M = 5000
    refused(vs, vs.VCSR_EINVAL, vs.run_rmsnorm_grad_gpu, dy=mat(M, 8), s=mat(M, 8), weight=mat(8),
            rstd=mat(M), dx=mat(M, 8), dweight=mat(8), workspace=ws)


LINEAR = {
    "w of another type": dict(w=bf(5, 8)),
    "w of another length": dict(w=mat(5, 9)),
    "y of another shape": dict(y=mat(4, 6)),
    "8-bit y": dict(y=f8(4, 5)),
    "8-bit without scales": dict(x=f8(4, 8), w=f8(5, 8)),
    "scales without 8-bit": dict(x_scale=mat(4), w_scale=mat(5)),
    "short w_scale": dict(x=f8(4, 8), w=f8(5, 8), x_scale=mat(4), w_scale=mat(4)),
    "short bias": dict(bias=mat(4)),
    "unknown activation": dict(act="tanh"),
    "residual of another type": dict(residual=bf(4, 5)),
    "z over y": dict(y=mat(4, 5, ptr=8192), z=mat(4, 5, ptr=8192)),
    "z over residual": dict(y=mat(4, 5, ptr=65536), z=mat(4, 5, ptr=8192),
                            residual=mat(4, 5, ptr=8192)),
    "residual over y of another stride": dict(y=mat(4, 5, ptr=8192),
                                              residual=mat(4, 5, ptr=8192, ld=9, nbytes=4096)),
    "misaligned w": dict(w=mat(5, 8, ptr=4099)),
    "no w": dict(w=mat(5, 8, ptr=0)),
    "short workspace": dict(x=mat(4, 4096), w=mat(5, 4096), workspace=f8(16)),
}


@pytest.mark.parametrize("case", LINEAR)
def test_linear_refuses(vs, case):
    kw = dict(x=mat(4, 8), w=mat(5, 8), y=mat(4, 5))
    kw.update(LINEAR[case])
    refused(vs, vs.VCSR_EINVAL, vs.run_linear_gpu, **kw)


def test_sizes_past_the_kernels_are_a_range_error(vs):
    lib = vs.load_library()
    a = vs._LinearArgs(M=1 << 31, N=4, K=4, x=4096, w=4096, y=4096)
    assert lib.vcsr_linear(C.byref(a), None, None) == vs.VCSR_ERANGE
    a = vs._LinearArgs(M=4, N=4, K=4, x=4096, w=4096, y=4096, ldx=(1 << 22) + 1)
    assert lib.vcsr_linear(C.byref(a), None, None) == vs.VCSR_ERANGE
    a = vs._RmsnormArgs(M=1 << 31, C=4, x=4096, weight=4096, y=8192)
    assert lib.vcsr_rmsnorm(C.byref(a), None, None) == vs.VCSR_ERANGE
    assert b"M" in lib.vcsr_last_error()
    a = vs._LinearArgs(M=(1 << 31) - 1, N=1 << 20, K=4, x=4096, w=4096, y=4096)
    assert lib.vcsr_linear(C.byref(a), None, None) == vs.VCSR_ERANGE


LINEAR_GRAD = {
    "no z for an activation": dict(act="gelu", dx=mat(4, 8)),
    "8-bit operands": dict(x=f8(4, 8), w=f8(5, 8), dx=f8(4, 8)),
    "z of another type": dict(act="relu", z=bf(4, 5), dx=mat(4, 8)),
    "dx of another type": dict(dx=bf(4, 8)),
    "dw of another shape": dict(dw=mat(8, 5)),
    "short dbias": dict(dbias=mat(4)),
    "short workspace": dict(act="relu", z=mat(4, 5), dx=mat(4, 8), workspace=f8(8)),
}


@pytest.mark.parametrize("case", LINEAR_GRAD)
def test_linear_grad_refuses(vs, case):
    kw = dict(dy=mat(4, 5), x=mat(4, 8), w=mat(5, 8))
    kw.update(LINEAR_GRAD[case])
    refused(vs, vs.VCSR_EINVAL, vs.run_linear_grad_gpu, **kw)


ADAMW = {
    "no grad": dict(grad=None),
    "param of bf16": dict(param=bf(300)),
    "8-bit grad": dict(grad=f8(300)),
    "bf16 states": dict(m=bf(300), v=bf(300)),
    "states of two types": dict(m=f8(300), m_scale=mat(2), v_scale=mat(2)),
    "8-bit states without scales": dict(m=f8(300), v=f8(300)),
    "short scales": dict(m=f8(300), v=f8(300), m_scale=mat(1), v_scale=mat(2)),
    "short v": dict(v=mat(299)),
    "copy of float32": dict(copy=mat(300)),
    "null param": dict(param=mat(300, ptr=0)),
    "misaligned grad": dict(grad=mat(300, ptr=4097)),
    "decay not finite": dict(weight_decay=float("inf")),
}


@pytest.mark.parametrize("case", ADAMW)
def test_adamw_refuses(vs, case):
    t = dict(param=mat(300), grad=mat(300), m=mat(300), v=mat(300))
    t.update(ADAMW[case])
    refused(vs, vs.VCSR_EINVAL, vs.AdamW, [t])


def test_null_arguments(vs):
    lib = vs.load_library()
    for fn in ("vcsr_rmsnorm", "vcsr_rmsnorm_grad", "vcsr_linear", "vcsr_linear_grad"):
        assert getattr(lib, fn)(None, None, None) == vs.VCSR_EINVAL, fn
    assert lib.vcsr_linear_workspace(None, None) == vs.VCSR_EINVAL
    assert lib.vcsr_adamw_step(None, None, None, None) == vs.VCSR_EINVAL
    assert lib.vcsr_adamw_create(None, 1, None, C.byref(C.c_void_p())) == vs.VCSR_EINVAL
    lib.vcsr_adamw_free(None)


def test_without_a_gpu_a_good_call_says_so(vs):
    if vs.device_count() > 0:
        pytest.skip("a GPU is visible")
    refused(vs, vs.VCSR_EDEVICE, vs.run_rmsnorm_gpu, mat(4, 8), mat(8), mat(4, 8, ptr=65536))
    refused(vs, vs.VCSR_EDEVICE, vs.run_linear_gpu, mat(4, 8), mat(5, 8), mat(4, 5))
