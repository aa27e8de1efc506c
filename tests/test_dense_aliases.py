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
