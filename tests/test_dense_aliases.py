"""Outputs over inputs that are refused before any device work (CPU)."""
from __future__ import annotations

import pytest

from test_dense_refusals import bf, mat, refused

A, B, D, E, F = (1 << 20 << i for i in range(5))

NORM_GRAD = {
    "dx over dsum of another stride": dict(dsum=mat(4, 8, ptr=A), dx=mat(4, 8, ptr=A, ld=9)),
    "dx over s of another stride": dict(s=mat(4, 8, ptr=A, ld=16), dx=mat(4, 8, ptr=A)),
    "dx over dy of another stride": dict(dy=mat(4, 8, ptr=A), dx=mat(4, 8, ptr=A, ld=12)),
    "dx over dy of another type": dict(dy=bf(4, 8, ptr=A), dx=mat(4, 8, ptr=A)),
}


@pytest.mark.parametrize("case", NORM_GRAD)
def test_rmsnorm_grad_refuses_shared_buffers(vs, case):
    kw = dict(dy=mat(4, 8, ptr=B), s=mat(4, 8, ptr=D), weight=mat(8), rstd=mat(4),
              dx=mat(4, 8, ptr=E))
    kw.update(NORM_GRAD[case])
    refused(vs, vs.VCSR_EINVAL, vs.run_rmsnorm_grad_gpu, **kw)


@pytest.mark.parametrize("over", ["dsum", "s", "dy"])
def test_rmsnorm_grad_takes_the_same_matrix(vs, over):
    """Passes the checks: without a GPU the device is what is missing."""
    if vs.device_count() > 0:
        pytest.skip("a GPU is visible")
    kw = dict(dy=mat(4, 8, ptr=B), s=mat(4, 8, ptr=D), dsum=mat(4, 8, ptr=A), weight=mat(8),
              rstd=mat(4))
    refused(vs, vs.VCSR_EDEVICE, vs.run_rmsnorm_grad_gpu, dx=kw[over], **kw)


LINEAR_GRAD = {
    "dx over dy": dict(dx=mat(8, 8, ptr=A)),
    "dx over w": dict(dx=mat(8, 8, ptr=D)),
    "dx over x, with dw": dict(dx=mat(8, 8, ptr=B), dw=mat(8, 8, ptr=E)),
    "dx over dw": dict(dx=mat(8, 8, ptr=E), dw=mat(8, 8, ptr=E)),
    "dw over dy": dict(dw=mat(8, 8, ptr=A)),
    "dw over x": dict(dw=mat(8, 8, ptr=B)),
    "dw over x, dz in the workspace": dict(dw=mat(8, 8, ptr=B), act="silu",
                                           z=mat(8, 8, ptr=F)),
    "dw over w, with dx": dict(dw=mat(8, 8, ptr=D), dx=mat(8, 8, ptr=E)),
}


@pytest.mark.parametrize("case", LINEAR_GRAD)
def test_linear_grad_refuses_outputs_over_operands(vs, case):
    kw = dict(dy=mat(8, 8, ptr=A), x=mat(8, 8, ptr=B), w=mat(8, 8, ptr=D),
              workspace=mat(1 << 20, ptr=1 << 30))
    kw.update(LINEAR_GRAD[case])
    refused(vs, vs.VCSR_EINVAL, vs.run_linear_grad_gpu, **kw)


@pytest.mark.parametrize("kw", [
    dict(dx=mat(8, 8, ptr=B)), dict(dw=mat(8, 8, ptr=D)),
    dict(dx=mat(8, 8, ptr=A), act="silu", z=mat(8, 8, ptr=F)),
    dict(dx=mat(8, 8, ptr=F), act="silu", z=mat(8, 8, ptr=F))],
    ids=["dx over x", "dw over w", "dx over dy", "dx over z"])
def test_linear_grad_takes_outputs_over_what_no_product_reads(vs, kw):
    """Passes the checks: without a GPU the device is what is missing."""
    if vs.device_count() > 0:
        pytest.skip("a GPU is visible")
    refused(vs, vs.VCSR_EDEVICE, vs.run_linear_grad_gpu, dy=mat(8, 8, ptr=A), x=mat(8, 8, ptr=B),
            w=mat(8, 8, ptr=D), workspace=mat(1 << 20, ptr=1 << 30), **kw)
