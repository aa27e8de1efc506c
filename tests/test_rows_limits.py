"""Widths at which the kernels for few rows would need 2^32 threads (CPU)."""
from __future__ import annotations

import pytest

from dense_plans import linear_plan
from gated_plans import gated_plan


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
