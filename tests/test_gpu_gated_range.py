"""The gated projection's gradient where dy * z_up alone passes FP32's range and dy * z_up *
act'(z_gate) does not, on the GPU."""
from __future__ import annotations

import numpy as np
import pytest

from block_ref import rounding, values
from dense_ref import EPS, Mat, act, act_grad, close, vector

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act_kind, z", [("relu", -1.0), ("silu", -30.0), ("gelu", -6.0),
                                         ("silu", -200.0), ("gelu", -50.0)])
@pytest.mark.parametrize("shape", [(1, 1, 1), (5, 3, 9), (70, 130, 65), (300, 64, 128)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("types", ["f32 f32", "bf16 bf16", "bf16 f32", "f32 bf16"])
def test_gated_grad_where_a_factor_is_small(gpu, types, shape, act_kind, z):
    xk, yk = types.split()
    vs, st = gpu, gpu.Stream()
    M, N, K = shape
    rng = np.random.default_rng(M + N)
    x, wg, wu = values(rng, (M, K), xk), values(rng, (N, K), xk), values(rng, (N, K), xk)
    dy, zu = values(rng, (M, N), yk), values(rng, (M, N), yk)
    zg = np.full((M, N), z)
    # 2^132 and more, in every row.
    dy, zu = (np.copysign(2.0 ** 66 * (1 + np.abs(v) % 1), v) for v in (dy, zu))
    dy, zu = (v.astype(np.float32).astype(np.float64) if yk == "f32"
              else vs.from_bf16(vs.to_bf16(v)).astype(np.float64) for v in (dy, zu))
    assert (np.abs(dy * zu) > np.finfo(np.float32).max).all()
    DX, DG = Mat(vs, st, None, xk, shape=(M, K)), Mat(vs, st, None, xk, shape=(N, K))
    DU = Mat(vs, st, None, xk, shape=(N, K))
    bg, bu = vector(vs, st, np.full(N, np.nan)), vector(vs, st, np.full(N, np.nan))
    print(f"gated grad range {types} {shape} {act_kind} {z}", flush=True)
    vs.run_gated_grad_gpu(Mat(vs, st, dy, yk).view, Mat(vs, st, x, xk).view,
                          Mat(vs, st, wg, xk).view, Mat(vs, st, wu, xk).view,
                          Mat(vs, st, zg, yk).view, Mat(vs, st, zu, yk).view, act=act_kind,
                          dx=DX.view, dw_gate=DG.view, dw_up=DU.view, dgate_bias=bg, dup_bias=bu,
                          stream=st)
    st.sync()
    with np.errstate(over="ignore"):
        dg, du = dy * zu * act_grad(zg, act_kind), dy * act(zg, act_kind)
    # The exponential's argument, at most 289 (silu at -200), is off by 3 u of itself, which
    # its value takes over; gelu's has four more roundings.  Where the value passes below
    # 2^-126 it may be zero: dz is off by 2^-126 of 2^134 then, the size that is left of it.
    rel = {"relu": 4, "silu": 4 * 289 + 40, "gelu": 8 * 289 + 40}[act_kind] * EPS
    eg, eu = rel * np.abs(dg) + 2.0 ** -126 * np.abs(dy * zu) * np.abs(z), \
        rel * np.abs(du) + 2.0 ** -126 * np.abs(dy * z)
    bias = (dg.sum(0), eg.sum(0) + (M + 4) * EPS * np.abs(dg).sum(0)), \
        (du.sum(0), eu.sum(0) + (M + 4) * EPS * np.abs(du).sum(0))
    if xk == "bf16":
        eg, eu = eg + rounding(dg, "bf16") * 1.01, eu + rounding(du, "bf16") * 1.01
    ag, au = np.abs(dg), np.abs(du)
    dx = dg @ wg + du @ wu
    tx = eg @ np.abs(wg) + eu @ np.abs(wu) + (2 * N + 6) * EPS * (ag @ np.abs(wg) + au @ np.abs(wu))
    close(DX.values(), dx, tx + rounding(dx, xk), "dx")
    for mat, d, e, a, name in ((DG, dg, eg, ag, "dw_gate"), (DU, du, eu, au, "dw_up")):
        want = d.T @ x
        tol = e.T @ np.abs(x) + (M + 4) * EPS * (a.T @ np.abs(x))
        close(mat.values(), want, tol + rounding(want, xk), name)
    for v, (want, tol), name in ((bg, bias[0], "dgate_bias"), (bu, bias[1], "dup_bias")):
        close(v.numpy(st), want, tol, name)
