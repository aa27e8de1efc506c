"""Widths at which the kernels for few rows would need 2^32 threads (CPU)."""
from __future__ import annotations

import pytest

from dense_plans import linear_plan
from gated_plans import gated_grad_plan, gated_plan


@pytest.mark.parametrize("N, tile16", [((1 << 27) - 16, True), ((1 << 27) - 15, False),
                                       ((1 << 27) - 1, False), (1 << 27, False)])
def test_linear_of_few_rows(vs, N, tile16):
    """16 columns a block of 512 threads: 2^23 blocks are too many."""
    assert (linear_plan(vs, 4, N, 4, "f32", "f32")[0] == 16) == tile16


@pytest.mark.parametrize("N, tile16", [((1 << 26) - 8, True), ((1 << 26) - 7, False),
                                       (1 << 26, False)])
def test_gated_of_few_rows(vs, N, tile16):
    """8 columns a block."""
    assert (gated_plan(vs, 4, N, 4, "f32", "f32")[0] == 16) == tile16


@pytest.mark.parametrize("what", [dict(dw=False), dict()], ids=["dx", "dx and dw"])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_gated_gradient_of_rows_in_one_launch(vs, kind, what):
    """dx has 2^24 - 1 tiles of 64 rows, which leave no block for dbias, or some fewer."""
    rows = 64 << 24
    assert gated_grad_plan(vs, rows - 64 - (64 << 18), 1, 64, kind, **what)[3:] == (64, 1)
    with pytest.raises(vs.VcsrError) as e:
        vs._gated_grad_bytes(rows - 64, 1, 64, {"f32": 0, "bf16": 1}[kind],
                             {"f32": 0, "bf16": 1}[kind], True, "dw" not in what, True, True)
    assert e.value.code == vs.VCSR_ERANGE
    assert gated_grad_plan(vs, rows, 1, 64, kind, **what)[3:] == (128, 1)
