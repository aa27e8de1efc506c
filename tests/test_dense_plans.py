"""The planner on the CPU: the sizes that the GPU tests run for a kernel choose it,
and a forced plan is what a product then takes."""
from __future__ import annotations

import pytest

from dense_plans import TILES, forced, grad_plan, linear_plan
from test_gpu_dense_kernels import GRAD_SIZES, LINEAR_SIZES


@pytest.mark.parametrize("size", LINEAR_SIZES, ids=lambda s: "x".join(map(str, s[:4])))
def test_forward_sizes(vs, size):
    got = linear_plan(vs, *size[:4], residual=True)
    assert all(w is None or g == w for g, w in zip(got, size[4])), got


@pytest.mark.parametrize("size", GRAD_SIZES, ids=lambda s: "x".join(map(str, s[:4])))
def test_gradient_sizes(vs, size):
    got = grad_plan(vs, *size[:4])
    assert all(w is None or g == w for g, w in zip(got, size[4])), got


def test_the_sizes_reach_every_large_kernel():
    """Between them: the 256 tile by rows and by columns, in a pair and alone, and
    dx and dw in launches of their own."""
    assert {s[3] for s in LINEAR_SIZES if s[4][0] == 256} == {"bf16", "fp8"}
    pairs = [s[4] for s in GRAD_SIZES if s[3] == "bf16"]
    assert any(p[0] and p[1] == 256 for p in pairs)
    assert any(not p[0] and p[1] == 256 for p in pairs)
    assert any(not p[0] and p[3] == 256 for p in pairs)


def test_forced_plans(vs):
    free = linear_plan(vs, 300, 300, 700, "bf16")
    for kind, tiles in TILES.items():
        for tile, stages in tiles:
            with forced(vs, tile, stages, splits=2):
                assert linear_plan(vs, 300, 300, 700, kind) == (tile, stages, 2, 300)
            with forced(vs, tile, stages, rows=tile):
                assert linear_plan(vs, 300, 300, 700, kind) == (tile, stages, 1, tile)
    with forced(vs, 256, together=True):
        assert grad_plan(vs, 300, 300, 700, "bf16") == (1, 256, 1, 256, 1)
        assert linear_plan(vs, 300, 300, 700, "f32")[0] != 256  # FP32 has none
    with forced(vs, 128, splits=3):
        assert grad_plan(vs, 300, 300, 700, "f32") == (0, 128, 3, 128, 3)
    assert linear_plan(vs, 300, 300, 700, "bf16") == free
