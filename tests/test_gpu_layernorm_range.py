"""Layer norm and its gradient where a factor of a row leaves FP32's range, on the GPU: what
lies behind a row's end must not reach its sums, nor a row another one."""
from __future__ import annotations

import numpy as np
import pytest

from block_ref import rounding, values
from dense_ref import EPS, Mat, close, vector

pytestmark = pytest.mark.gpu


# Rows that end in a lane's vector and before its first, that fill their lanes, and of
# every kernel: a thread a row, groups of lanes, one wave and several a row, read twice.
@pytest.mark.parametrize("C", [1, 3, 6, 8, 20, 64, 100, 200, 256, 330, 515, 1000, 2050, 4096, 5000,
                               8190, 9001, 17001])
@pytest.mark.parametrize("kinds", ["f32 f32", "bf16 bf16", "f32 bf16", "bf16 f32"])
def test_layernorm_grad_of_constant_rows_far_from_zero(gpu, kinds, C):
    """s = mean = 2^120 and rstd = 1 / sqrt(1e-5): h is zero, mean * rstd past FP32.  With h
    = 0, dx = dsum + rstd * (g - mean(g)) and dweight has nothing of such a row."""
    xk, yk = kinds.split()
    vs, st, rng = gpu, gpu.Stream(), np.random.default_rng(C)
    M, far = 7, np.array([0, 2, 6])
    s, dy, dsum = values(rng, (M, C), xk), values(rng, (M, C), yk), values(rng, (M, C), xk)
    mean, rstd = 0.1 * rng.standard_normal(M), 0.5 + rng.random(M)
    s[far] = 2.0 ** 120
    mean[far], rstd[far] = 2.0 ** 120, 1e-5 ** -0.5
    mean, rstd = mean.astype(np.float32), rstd.astype(np.float32)
    assert (mean[far].astype(np.float64) * rstd[far] > np.finfo(np.float32).max).all()
    w = (1 + 0.2 * rng.standard_normal(C)).astype(np.float32).astype(np.float64)
    DX = Mat(vs, st, None, xk, shape=(M, C))
    dweight, dbias = vector(vs, st, np.full(C, np.nan)), vector(vs, st, np.full(C, np.nan))
    print(f"layernorm grad far {kinds} C={C}", flush=True)
    vs.run_layernorm_grad_gpu(Mat(vs, st, dy, yk).view, Mat(vs, st, s, xk).view,
                              vector(vs, st, w), vector(vs, st, mean), vector(vs, st, rstd),
                              DX.view, dweight, dbias, dsum=Mat(vs, st, dsum, xk).view, stream=st)
    st.sync()
    mu, r = (v.astype(np.float64)[:, None] for v in (mean, rstd))
    h, g = (s - mu) * r, dy * w
    mg, mgh = g.mean(1, keepdims=True), (g * h).mean(1, keepdims=True)
    dx = dsum + r * (g - mg - h * mgh)
    # Chains of at most C terms for a row's sums and M for a column's, some roundings each.
    ag, ah = np.abs(g), np.abs(h)
    sg, sgh = ag.mean(1, keepdims=True), (ag * ah).mean(1, keepdims=True)
    tol = r * ((C + 6) * EPS * (sg + ah * sgh) + 8 * EPS * (ag + sg + ah * sgh)) + 8 * EPS * np.abs(dx)
    close(DX.values(), dx, tol + rounding(dx, xk), f"dx {kinds} {C}")
    close(dweight.numpy(st), (dy * h).sum(0), (M + 8) * EPS * (np.abs(dy) * ah).sum(0) + 1e-30,
          f"dweight {kinds} {C}")
    close(dbias.numpy(st), dy.sum(0), (M + 4) * EPS * np.abs(dy).sum(0) + 1e-30, f"dbias {kinds} {C}")


@pytest.mark.parametrize("yk", ["f32", "bf16", "fp8"])
@pytest.mark.parametrize("C", [2, 64, 100, 700, 9001])
def test_layernorm_of_squares_below_fp32(gpu, C, yk):
    """Deviations of 2^-80, whose squares are zero in FP32: beside eps they count for nothing,
    without it rstd is infinite and y infinite or NaN, in that row alone."""
    vs, st, rng = gpu, gpu.Stream(), np.random.default_rng(C)
    x = values(rng, (3, C), "f32")
    x[1] = 2.0 ** -80 * np.where(np.arange(C) % 2, 1, -1)
    b = (0.3 * rng.standard_normal(C)).astype(np.float32)
    for eps in (1e-5, 1e-12, 0.0):
        Y, rstd = Mat(vs, st, None, yk, shape=(3, C)), vector(vs, st, np.zeros(3))
        scale = vector(vs, st, np.zeros(3)) if yk == "fp8" else None
        print(f"layernorm tiny {yk} C={C} eps={eps}", flush=True)
        vs.run_layernorm_gpu(Mat(vs, st, x, "f32").view, vector(vs, st, np.ones(C)), Y.view,
                             bias=vector(vs, st, b), rstd=rstd, y_scale=scale, eps=eps, stream=st)
        st.sync()
        y, r = Y.values(), rstd.numpy(st)
        if yk == "fp8":
            with np.errstate(invalid="ignore"):
                y = y * scale.numpy(st).astype(np.float64)[:, None]
        assert np.isfinite(y[[0, 2]]).all() and np.isfinite(r[[0, 2]]).all()
        if eps:
            # (t - mean) * rstd is at most 2^-80 * 1e6, less than any bias' rounding.
            want = b.astype(np.float64)
            tol = 2 * EPS * np.abs(want) + 2.0 ** -59 + rounding(want, "f32" if yk == "fp8" else yk)
            if yk == "fp8":  # codes of b / scale, the scale from the largest
                tol += np.maximum(2.0 ** -4 * np.abs(want), 2.0 ** -10 * np.abs(want).max() / 448)
            close(y[1], want, tol * 1.01, f"{yk} {C} {eps}")
        else:
            assert np.isinf(r[1]) and not np.isfinite(y[1]).any()
