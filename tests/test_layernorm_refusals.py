"""Arguments layer norm and its gradient refuse, before any device work (CPU)."""
from __future__ import annotations

import ctypes as C

import pytest

from test_dense_refusals import Fake, bf, f8, mat, refused

A, B, D, E = (1 << 20 << i for i in range(4))

NORM = {
    "y of another shape": dict(y=mat(4, 7)),
    "8-bit x": dict(x=f8(4, 8)),
    "x of no known type": dict(x=Fake((4, 8), "int32")),
    "residual of another type": dict(residual=bf(4, 8)),
    "sum of another type": dict(sum=bf(4, 8)),
    "no weight": dict(weight=mat(8, ptr=0)),
    "short weight": dict(weight=mat(7)),
    "short bias": dict(bias=mat(7)),
    "bias of bf16": dict(bias=bf(8)),
    "misaligned bias": dict(bias=mat(8, ptr=4098)),
    "short mean": dict(mean=mat(3)),
    "misaligned mean": dict(mean=mat(4, ptr=4097)),
    "mean over rstd": dict(mean=mat(4, ptr=A), rstd=mat(4, ptr=A)),
    "misaligned rstd": dict(rstd=mat(4, ptr=4097)),
    "stride under the row": dict(x=mat(4, 8, ld=6, nbytes=4096)),
    "x too short for its stride": dict(x=mat(4, 8, ld=64, nbytes=128)),
    "negative eps": dict(eps=-1e-6),
    "eps not finite": dict(eps=float("inf")),
    "8-bit y without scales": dict(y=f8(4, 8)),
    "scales without 8-bit y": dict(y_scale=mat(4)),
    "short scales": dict(y=f8(4, 8), y_scale=mat(3)),
    "no x": dict(x=mat(4, 8, ptr=0)),
    "no y": dict(y=mat(4, 8, ptr=0)),
    "misaligned x": dict(x=mat(4, 8, ptr=4098)),
    "y over x of another type": dict(x=mat(4, 8, ptr=A), y=bf(4, 8, ptr=A)),
    "y over residual of another stride": dict(residual=mat(4, 8, ptr=A),
                                              y=mat(4, 8, ptr=A, ld=9)),
    "sum over y": dict(sum=mat(4, 8, ptr=65536)),
    "sum over x of another stride": dict(x=mat(4, 8, ptr=A), sum=mat(4, 8, ptr=A, ld=9)),
    "no columns": dict(x=mat(4, 0), y=mat(4, 0), weight=mat(0)),
}


@pytest.mark.parametrize("case", NORM)
def test_layernorm_refuses(vs, case):
    kw = dict(x=mat(4, 8), weight=mat(8), y=mat(4, 8, ptr=65536))
    kw.update(NORM[case])
    refused(vs, vs.VCSR_EINVAL, vs.run_layernorm_gpu, **kw)


GRAD = {
    "dy of another shape": dict(dy=mat(4, 9)),
    "8-bit dy": dict(dy=f8(4, 8)),
    "dx of another type": dict(dx=bf(4, 8)),
    "no rstd": dict(rstd=None),
    "no mean": dict(mean=None),
    "short mean": dict(mean=mat(3)),
    "misaligned dbias": dict(dbias=mat(8, ptr=4098)),
    "dbias over dweight": dict(dweight=mat(8, ptr=8192), dbias=mat(8, ptr=8192)),
    "dx over dsum of another stride": dict(dsum=mat(4, 8, ptr=A), dx=mat(4, 8, ptr=A, ld=9)),
    "dx over s of another stride": dict(s=mat(4, 8, ptr=A, ld=16), dx=mat(4, 8, ptr=A)),
    "dx over dy of another type": dict(dy=bf(4, 8, ptr=A), dx=mat(4, 8, ptr=A)),
}


@pytest.mark.parametrize("case", GRAD)
def test_layernorm_grad_refuses(vs, case):
    kw = dict(dy=mat(4, 8, ptr=B), s=mat(4, 8, ptr=D), weight=mat(8), mean=mat(4), rstd=mat(4),
              dx=mat(4, 8, ptr=E))
    kw.update(GRAD[case])
    refused(vs, vs.VCSR_EINVAL, vs.run_layernorm_grad_gpu, **kw)


@pytest.mark.parametrize("ws", [f8(16), f8(1 << 20, ptr=4104)], ids=["short", "misaligned"])
@pytest.mark.parametrize("sums", ["dweight", "dbias"])
def test_layernorm_grad_refuses_a_workspace(vs, ws, sums):
    """Many rows: the sums go through partial rows."""
    M = 5000
    refused(vs, vs.VCSR_EINVAL, vs.run_layernorm_grad_gpu, dy=mat(M, 8), s=mat(M, 8), weight=mat(8),
            mean=mat(M), rstd=mat(M), dx=mat(M, 8), workspace=ws, **{sums: mat(8)})


def test_layernorm_grad_workspace_goes_by_its_sums(vs):
    one = vs._layernorm_grad_bytes(5000, 130, 0, 0, True, False)
    assert one > 0 and vs._layernorm_grad_bytes(5000, 130, 0, 0, False, True) == one
    assert vs._layernorm_grad_bytes(5000, 130, 0, 0, True, True) == 2 * one
    assert vs._layernorm_grad_bytes(5000, 130, 0, 0, False, False) == 0
    assert vs._layernorm_grad_bytes(0, 130, 0, 0, True, True) == 0


def test_layernorm_null_arguments_and_sizes(vs):
    lib = vs.load_library()
    for fn in ("vcsr_layernorm", "vcsr_layernorm_grad"):
        assert getattr(lib, fn)(None, None, None) == vs.VCSR_EINVAL, fn
    assert lib.vcsr_layernorm_grad_workspace(None, None) == vs.VCSR_EINVAL
    a = vs._LayernormArgs(M=1 << 31, C=4, x=4096, weight=4096, y=8192)
    assert lib.vcsr_layernorm(C.byref(a), None, None) == vs.VCSR_ERANGE
    a = vs._LayernormArgs(M=-1, C=4, x=4096, weight=4096, y=8192)
    assert lib.vcsr_layernorm(C.byref(a), None, None) == vs.VCSR_EINVAL


def test_layernorm_without_a_gpu_says_so(vs):
    if vs.device_count() > 0:
        pytest.skip("a GPU is visible")
    refused(vs, vs.VCSR_EDEVICE, vs.run_layernorm_gpu, mat(4, 8), mat(8), mat(4, 8, ptr=65536))
    for over in (B, D, E):  # dx over dy or s passes the checks
        refused(vs, vs.VCSR_EDEVICE, vs.run_layernorm_grad_gpu, mat(4, 8, ptr=B), mat(4, 8, ptr=D),
                mat(8), mat(4), mat(4), mat(4, 8, ptr=over))
