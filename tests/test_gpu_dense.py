"""The dense operators on the GPU against their formulas in 64 bits.

Tolerances, all set before a first run: u = 2^-24.  A sum of n products in
FP32 in any order is off by at most (n + 2) u times the sum of magnitudes; the
RMS factor by (C / 8 + 16) u at worst (its sum of squares is added in chains of
at most C / 8 terms); a rounding to bf16 (8 significant bits) adds 2^-8 relative, to e4m3 2^-4 (or
half its smallest step, 2^-10)."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from conftest import capture, hip_runtime
from dense_ref import (E4M3, EPS, NP, ROUND, TINY, Mat, act, act_grad, close, from_fp8, pack,
                       rms_norm, rms_norm_grad, unpack, vector)

pytestmark = pytest.mark.gpu


def values(rng, shape, kind, scale=1.0):
    """Random values that `kind` holds exactly."""
    return unpack(pack(scale * rng.standard_normal(shape), kind), kind)


def rounding(v, kind):
    return np.abs(v) * ROUND[kind] + TINY[kind]


# -------------------------------------------------------------------- RMS norm
def norm_once(vs, st, x, r, w, xk, yk, eps, pad=0, off=0, with_sum=True):
    M, C = x.shape
    X = Mat(vs, st, x, xk, pad, off)
    R = Mat(vs, st, r, xk, pad, 2 * off) if r is not None else None
    S = Mat(vs, st, None, xk, pad, off, (M, C)) if with_sum else None
    Y = Mat(vs, st, None, yk, pad, off, (M, C))
    scale = vector(vs, st, np.zeros(M)) if yk == "fp8" else None
    rstd = vector(vs, st, np.zeros(M))
    dw = vector(vs, st, w)
    vs.run_rmsnorm_gpu(X.view, dw, Y.view, residual=R.view if R else None,
                       sum=S.view if S else None, y_scale=scale, rstd=rstd, eps=eps, stream=st)
    st.sync()
    X.codes()
    return Y, S, scale.numpy(st) if scale else None, rstd.numpy(st)


def check_norm(vs, st, x, r, w, xk, yk, eps, what, **kw):
    C = x.shape[1]
    Y, S, scale, rstd = norm_once(vs, st, x, r, w, xk, yk, eps, **kw)
    with np.errstate(all="ignore"):
        t, want_rstd, want = rms_norm(x, r, w, eps)
    u = (C / 8 + 16) * EPS
    close(rstd, want_rstd[:, 0], np.abs(want_rstd[:, 0]) * u, what + " rstd")
    if S:
        close(S.values(), t, rounding(t, xk) + np.abs(t) * EPS, what + " sum")
    if yk == "fp8":
        with np.errstate(all="ignore"):
            top = np.max(np.abs(want), axis=1)
            want_scale = np.where(top < 1e-30, 1e-30, top) / 448
        close(scale, want_scale, want_scale * (u + 4 * EPS), what + " scale")
        with np.errstate(all="ignore"):
            q = want / want_scale[:, None]
        close(Y.values(), q, np.maximum(np.abs(q) * (2.0 ** -4 + 2 * u), 2.0 ** -10), what)
    else:
        close(Y.values(), want, np.abs(want) * (u + 4 * EPS) + rounding(want, yk), what)


@pytest.mark.parametrize("C", [1, 3, 8, 31, 64, 128, 130, 257, 512, 1000, 2050, 4096, 8191, 9001])
@pytest.mark.parametrize("kinds", ["f32 f32", "f32 bf16", "f32 fp8", "bf16 f32", "bf16 bf16",
                                   "bf16 fp8"])
def test_rmsnorm(gpu, kinds, C):
    xk, yk = kinds.split()
    st = gpu.Stream()
    rng = np.random.default_rng(C)
    for M, pad, off, residual in ((1, 0, 0, True), (5, 3, 1, True), (67, 0, 0, False)):
        print(f"rmsnorm {kinds} C={C} M={M} pad={pad} off={off}", flush=True)
        x = values(rng, (M, C), xk, 2.0)
        r = values(rng, (M, C), xk) if residual else None
        w = 1 + 0.2 * rng.standard_normal(C)
        w = w.astype(np.float32).astype(np.float64)
        check_norm(gpu, st, x, r, w, xk, yk, 1e-6, f"{kinds} {M}x{C}", pad=pad, off=off)


@pytest.mark.parametrize("kinds", ["f32 f32", "bf16 bf16", "bf16 fp8", "f32 fp8"])
@pytest.mark.parametrize("C", [40, 700, 12000])
def test_rmsnorm_rows_that_are_zero_or_not_finite(gpu, kinds, C):
    """A row of zeros, of tiny and of huge values, and rows with a NaN or an
    infinity, which reach no other row."""
    xk, yk = kinds.split()
    st = gpu.Stream()
    rng = np.random.default_rng(C)
    x = values(rng, (9, C), xk)
    x[1] = 0
    x[2] *= 2.0 ** -60
    x[3] *= 2.0 ** 50
    x[4, C // 2] = np.nan
    x[5, C - 1] = np.inf
    x[6, 0] = -np.inf
    w = np.ones(C)
    w[C // 3] = 0
    print(f"rmsnorm edge rows {kinds} C={C}", flush=True)
    check_norm(gpu, st, x, None, w, xk, yk, 1e-12, f"{kinds} edge rows", with_sum=False)


def test_rmsnorm_in_place(gpu):
    """sum over x and over the residual, y over x: the same bits as apart."""
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(5)
    for C in (100, 2000, 20000):
        x, r = values(rng, (7, C), "f32"), values(rng, (7, C), "f32")
        w = vector(vs, st, 1 + 0.1 * rng.standard_normal(C))
        X, R = Mat(vs, st, x, "f32"), Mat(vs, st, r, "f32")
        S, Y = Mat(vs, st, None, "f32", shape=(7, C)), Mat(vs, st, None, "f32", shape=(7, C))
        vs.run_rmsnorm_gpu(X.view, w, Y.view, residual=R.view, sum=S.view, stream=st)
        s, y = S.codes(), Y.codes()
        for into in ("x", "residual"):
            X, R = Mat(vs, st, x, "f32"), Mat(vs, st, r, "f32")
            Y = Mat(vs, st, None, "f32", shape=(7, C))
            D = X if into == "x" else R
            vs.run_rmsnorm_gpu(X.view, w, Y.view, residual=R.view, sum=D.view, stream=st)
            assert D.codes().tobytes() == s.tobytes() and Y.codes().tobytes() == y.tobytes(), into
        X, R = Mat(vs, st, x, "f32"), Mat(vs, st, r, "f32")
        vs.run_rmsnorm_gpu(X.view, w, X.view, residual=R.view, stream=st)
        assert X.codes().tobytes() == y.tobytes()


@pytest.mark.parametrize("C", [1, 7, 64, 130, 600, 2050, 8191, 9001])
@pytest.mark.parametrize("kinds", ["f32 f32", "bf16 bf16", "f32 bf16", "bf16 f32"])
def test_rmsnorm_grad(gpu, kinds, C):
    xk, yk = kinds.split()
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(100 + C)
    for M, pad, off, stream_grad in ((1, 0, 0, True), (6, 5, 1, False), (1500, 0, 0, True)):
        if M * C > 4e6:
            M = 300
        print(f"rmsnorm grad {kinds} C={C} M={M}", flush=True)
        s, dy = values(rng, (M, C), xk, 1.5), values(rng, (M, C), yk)
        ds = values(rng, (M, C), xk) if stream_grad else None
        w = (1 + 0.2 * rng.standard_normal(C)).astype(np.float32).astype(np.float64)
        rstd = (1 / np.sqrt(np.mean(s * s, axis=1) + 1e-6)).astype(np.float32)
        S, DY = Mat(vs, st, s, xk, pad, off), Mat(vs, st, dy, yk, pad, off)
        DS = Mat(vs, st, ds, xk, pad, off) if stream_grad else None
        DX = Mat(vs, st, None, xk, pad, off, (M, C))
        dweight = vector(vs, st, np.full(C, np.nan))
        vs.run_rmsnorm_grad_gpu(DY.view, S.view, vector(vs, st, w), vector(vs, st, rstd), DX.view,
                                dweight, dsum=DS.view if DS else None, stream=st)
        st.sync()
        rd = rstd.astype(np.float64)[:, None]
        want, want_w = rms_norm_grad(dy, s, w, rd, ds)
        h, g = np.abs(s * rd), np.abs(dy * w)
        dot = np.sum(g * h, axis=1, keepdims=True) / C
        tol = 8 * EPS * (rd * (g + h * dot) + np.abs(want)) + rd * h * dot * (C + 4) * EPS
        close(DX.values(), want, tol + rounding(want, xk), f"dx {kinds} {M}x{C}")
        close(dweight.numpy(st), want_w, (M + 6) * EPS * np.sum(np.abs(dy) * h, axis=0) + 1e-30,
              "dweight")


def test_rmsnorm_grad_against_differences(gpu):
    """The directional derivative of <dy, y> along a random direction, by central
    differences of the formula, against the kernel's gradients."""
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(9)
    M, C = 5, 96
    x, dy = values(rng, (M, C), "f32"), values(rng, (M, C), "f32")
    w = (1 + 0.2 * rng.standard_normal(C)).astype(np.float32).astype(np.float64)
    _, rstd, _ = rms_norm(x, None, w, 1e-6)
    X, DY, DX = (Mat(vs, st, x, "f32"), Mat(vs, st, dy, "f32"),
                 Mat(vs, st, None, "f32", shape=(M, C)))
    dweight = vector(vs, st, np.zeros(C))
    vs.run_rmsnorm_grad_gpu(DY.view, X.view, vector(vs, st, w), vector(vs, st, rstd[:, 0]),
                            DX.view, dweight, stream=st)
    st.sync()
    vx, vw, h = rng.standard_normal((M, C)), rng.standard_normal(C), 1e-5

    def loss(t):
        return np.sum(dy * rms_norm(x + t * vx, None, w + t * vw, 1e-6)[2])

    diff = (loss(h) - loss(-h)) / (2 * h)
    got = np.sum(DX.values() * vx) + np.sum(dweight.numpy(st).astype(np.float64) * vw)
    # Differences are good to h^2 and 2^-52 / h; the gradients to 2^-20 of their terms.
    size = np.sum(np.abs(DX.values() * vx)) + np.sum(np.abs(vw) * np.abs(dweight.numpy(st)))
    assert abs(diff - got) <= 2.0 ** -20 * size + 1e-8 * size


# ---------------------------------------------------------------------- linear
def linear_once(vs, st, rng, M, N, K, xk, yk, kind, pad=0, off=0, residual=True, bias=True,
                with_z=False):
    x, w = values(rng, (M, K), xk), values(rng, (N, K), xk, K ** -0.5)
    xs = ws = None
    if xk == "fp8":
        xs = (0.5 + rng.random(M)).astype(np.float32)
        ws = (0.5 + rng.random(N)).astype(np.float32)
    b = (0.3 * rng.standard_normal(N)).astype(np.float32) if bias else None
    r = values(rng, (M, N), yk) if residual else None
    X, W = Mat(vs, st, x, xk, pad, off), Mat(vs, st, w, xk, pad, off)
    Y = Mat(vs, st, None, yk, pad, off, (M, N))
    Z = Mat(vs, st, None, yk, pad, off, (M, N)) if with_z else None
    R = Mat(vs, st, r, yk, pad, off) if residual else None
    vs.run_linear_gpu(X.view, W.view, Y.view, bias=vector(vs, st, b) if bias else None,
                      residual=R.view if R else None, act=kind, z=Z.view if Z else None,
                      x_scale=vector(vs, st, xs) if xs is not None else None,
                      w_scale=vector(vs, st, ws) if ws is not None else None, stream=st)
    st.sync()
    xd, wd = (x, w) if xs is None else (x * xs.astype(np.float64)[:, None],
                                        w * ws.astype(np.float64)[:, None])
    z = xd @ wd.T + (b.astype(np.float64) if bias else 0)
    tz = (K + 4) * EPS * (np.abs(xd) @ np.abs(wd).T + (np.abs(b) if bias else 0))
    if with_z:
        close(Z.values(), z, tz + rounding(z, yk), "z")
    y = act(z, kind)
    # Each act's slope is at most 1.13; its own arithmetic is good to 16 u.
    ty = 1.13 * tz + 16 * EPS * np.abs(z)
    if residual:
        y = y + r
        ty = ty + EPS * np.abs(y)
    close(Y.values(), y, ty + rounding(y, yk), f"y {M}x{N}x{K} {xk} {yk} {kind}")
    return Y.codes()


SHAPES = [(1, 1, 1), (1, 64, 64), (3, 5, 7), (16, 33, 65), (17, 129, 40), (64, 64, 128),
          (65, 63, 130), (129, 200, 257), (300, 47, 514), (1, 1000, 4100), (9, 260, 2051),
          (130, 300, 1030)]


@pytest.mark.parametrize("types", ["f32 f32", "f32 bf16", "bf16 bf16", "bf16 f32", "fp8 bf16",
                                   "fp8 f32"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_linear(gpu, shape, types):
    xk, yk = types.split()
    st = gpu.Stream()
    rng = np.random.default_rng(sum(shape))
    for n, (kind, pad, off) in enumerate((("gelu", 0, 0), ("silu", 1, 1), ("relu", 16, 0),
                                          ("none", 8, 3))):
        print(f"linear {types} {shape} {kind} pad={pad} off={off}", flush=True)
        linear_once(gpu, st, rng, *shape, xk, yk, kind, pad, off, residual=n % 2 == 0,
                    bias=n != 3, with_z=n < 2)


@pytest.mark.parametrize("types", ["f32 f32", "bf16 bf16", "fp8 bf16"])
@pytest.mark.parametrize("shape", [(2048, 2048, 192), (4099, 1030, 96), (700, 4096, 640),
                                   (2500, 1000, 72), (513, 8200, 256),
                                   (7956, 2048, 1024), (5001, 4096, 512)],
                         ids=lambda s: "x".join(map(str, s)))
def test_linear_many_tiles(gpu, shape, types):
    """Sizes that fill the chip, whole and ragged."""
    xk, yk = types.split()
    st = gpu.Stream()
    print(f"linear {types} {shape}", flush=True)
    linear_once(gpu, st, np.random.default_rng(3), *shape, xk, yk, "silu", with_z=True)


@pytest.mark.parametrize("types", ["f32 f32", "bf16 f32"])
def test_linear_keeps_nan_and_infinity_in_their_rows(gpu, types):
    xk, yk = types.split()
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(4)
    for M, N, K in ((5, 40, 100), (200, 150, 70)):
        x, w = values(rng, (M, K), xk), np.abs(values(rng, (N, K), xk)) + 0.5
        w = unpack(pack(w, xk), xk)
        x[1, K - 1], x[2, 0], x[3, K // 2] = np.nan, np.inf, -np.inf
        with np.errstate(all="ignore"):
            y = x @ w.T
        Y = Mat(vs, st, None, yk, shape=(M, N))
        vs.run_linear_gpu(Mat(vs, st, x, xk).view, Mat(vs, st, w, xk).view, Y.view, stream=st,
                          act="relu")
        st.sync()
        with np.errstate(all="ignore"):
            tol = (K + 4) * EPS * (np.abs(np.nan_to_num(x, posinf=0, neginf=0)) @ w.T)
        close(Y.values(), act(y, "relu"), tol, f"{types} {M}x{N}x{K}")


def grad_once(vs, st, rng, M, N, K, xk, yk, kind, pad=0, off=0, want=("dx", "dw", "dbias")):
    x, w = values(rng, (M, K), xk), values(rng, (N, K), xk, K ** -0.5)
    z, dy = values(rng, (M, N), yk), values(rng, (M, N), yk)
    X, W = Mat(vs, st, x, xk, pad, off), Mat(vs, st, w, xk, pad, off)
    Z, DY = Mat(vs, st, z, yk, pad, off), Mat(vs, st, dy, yk, pad, off)
    DX, DW = Mat(vs, st, None, xk, pad, off, (M, K)), Mat(vs, st, None, xk, pad, off, (N, K))
    db = vector(vs, st, np.full(N, np.nan))
    vs.run_linear_grad_gpu(DY.view, X.view, W.view, z=Z.view, act=kind,
                           dx=DX.view if "dx" in want else None,
                           dw=DW.view if "dw" in want else None,
                           dbias=db if "dbias" in want else None, stream=st)
    st.sync()
    dz = dy * act_grad(z, kind)
    # act' is at most 1.13 in size and good to 32 u there.
    edz = 40 * EPS * np.abs(dy) * 1.13
    if "dbias" in want:
        close(db.numpy(st), dz.sum(0), edz.sum(0) + (M + 4) * EPS * np.abs(dz).sum(0), "dbias")
    if xk == "bf16":  # dz is an operand of the products
        edz = edz + rounding(dz, "bf16") * 1.01
    what = f"{M}x{N}x{K} {xk} {yk} {kind}"
    if "dx" in want:
        v = dz @ w
        tol = edz @ np.abs(w) + (N + 4) * EPS * (np.abs(dz) @ np.abs(w))
        close(DX.values(), v, tol + rounding(v, xk), "dx " + what)
    if "dw" in want:
        v = dz.T @ x
        tol = edz.T @ np.abs(x) + (M + 4) * EPS * (np.abs(dz).T @ np.abs(x))
        close(DW.values(), v, tol + rounding(v, xk), "dw " + what)


@pytest.mark.parametrize("types", ["f32 f32", "bf16 bf16", "bf16 f32", "f32 bf16"])
@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 64, 96), (3, 5, 7), (33, 65, 31), (64, 128, 64),
                                   (100, 130, 70), (500, 47, 260), (2100, 40, 136),
                                   (1000, 300, 520)], ids=lambda s: "x".join(map(str, s)))
def test_linear_grad(gpu, shape, types):
    xk, yk = types.split()
    st = gpu.Stream()
    rng = np.random.default_rng(sum(shape))
    for kind, pad, off in (("gelu", 0, 0), ("silu", 8, 0), ("relu", 3, 1), ("none", 0, 0)):
        print(f"linear grad {types} {shape} {kind} pad={pad} off={off}", flush=True)
        grad_once(gpu, st, rng, *shape, xk, yk, kind, pad, off)
    for want in (("dx",), ("dw",), ("dbias",)):
        grad_once(gpu, st, rng, *shape, xk, yk, "silu", want=want)


@pytest.mark.parametrize("types", ["f32 f32", "bf16 bf16"])
def test_linear_grad_many_tiles(gpu, types):
    xk, yk = types.split()
    for shape in ((2048, 2048, 256), (4100, 264, 2200)):
        print(f"linear grad {types} {shape}", flush=True)
        grad_once(gpu, gpu.Stream(), np.random.default_rng(8), *shape, xk, yk, "gelu")


def test_linear_grad_against_differences(gpu):
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(19)
    M, N, K = 6, 20, 24
    for kind in ("gelu", "silu", "none"):
        x, w = values(rng, (M, K), "f32"), values(rng, (N, K), "f32", 0.3)
        b, dy = 0.1 * rng.standard_normal(N), values(rng, (M, N), "f32")
        Z = Mat(vs, st, x @ w.T + b, "f32")
        DX = Mat(vs, st, None, "f32", shape=(M, K))
        DW, db = Mat(vs, st, None, "f32", shape=(N, K)), vector(vs, st, np.zeros(N))
        vs.run_linear_grad_gpu(Mat(vs, st, dy, "f32").view, Mat(vs, st, x, "f32").view,
                               Mat(vs, st, w, "f32").view, z=Z.view, act=kind, dx=DX.view,
                               dw=DW.view, dbias=db, stream=st)
        st.sync()
        vx, vw, vb = (rng.standard_normal(s) for s in ((M, K), (N, K), (N,)))
        h = 1e-5

        def loss(t):
            return np.sum(dy * act((x + t * vx) @ (w + t * vw).T + b + t * vb, kind))

        parts = (DX.values() * vx, DW.values() * vw, db.numpy(st).astype(np.float64) * vb)
        got, size = sum(p.sum() for p in parts), sum(np.abs(p).sum() for p in parts)
        assert abs((loss(h) - loss(-h)) / (2 * h) - got) <= (2.0 ** -19 + 1e-8) * size, kind


# ----------------------------------------------------------------------- AdamW
HYPER = dict(lr=3e-3, beta1=0.9, beta2=0.95, eps=1e-8, grad_scale=0.5)


def adamw_formula(p, g, m, v, decay, step):
    h = HYPER
    g = g * h["grad_scale"]
    m = h["beta1"] * m + (1 - h["beta1"]) * g
    v = h["beta2"] * v + (1 - h["beta2"]) * g * g
    mh, vh = m / (1 - h["beta1"] ** step), v / (1 - h["beta2"] ** step)
    return p - h["lr"] * (mh / (np.sqrt(vh) + h["eps"]) + decay * p), m, v


def blocks_of(n):
    return np.arange(n) // 256


@pytest.mark.parametrize("gk", ["f32", "bf16"])
def test_adamw_f32_states(gpu, gk):
    """Three steps over tensors of many sizes at once, one of them empty."""
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(31)
    sizes = [1, 3, 0, 255, 256, 257, 4095, 4096, 4097, 20000, 5]
    tensors, host = [], []
    for i, n in enumerate(sizes):
        off = i % 3
        p, g = values(rng, (1, n), "f32"), values(rng, (1, n), gk, 1e-2)
        if n > 4:
            g[0, 2] = 0.0
        d = dict(param=Mat(vs, st, p, "f32", off=off), grad=Mat(vs, st, g, gk, off=off),
                 m=Mat(vs, st, np.zeros((1, n)), "f32", off=off),
                 v=Mat(vs, st, np.zeros((1, n)), "f32", off=off))
        if i % 2:
            d["copy"] = Mat(vs, st, None, "bf16", off=off, shape=(1, n))
        tensors.append(d)
        host.append([p, g, np.zeros((1, n)), np.zeros((1, n)), 0.1 * (i % 2)])
    print(f"adamw f32 states, {gk} gradients", flush=True)
    opt = vs.AdamW([dict({k: m.view for k, m in d.items()}, weight_decay=h[4])
                    for d, h in zip(tensors, host)], stream=st)
    for step in (1, 2, 3):
        opt.step(step, stream=st, **HYPER)
        st.sync()
        for d, h in zip(tensors, host):
            p, m, v = adamw_formula(h[0], h[1], h[2], h[3], h[4], step)
            # A step's operations round a handful of times: 16 u of each term.
            move = np.abs(p - h[0]) + HYPER["lr"] * h[4] * np.abs(h[0])
            got_p = d["param"].values()
            close(got_p, p, 2 * EPS * np.abs(p) + 2 * EPS * np.abs(h[0]) + 24 * EPS * move, "param")
            close(d["m"].values(), m, 8 * EPS * (np.abs(h[2]) + np.abs(h[1])) + TINY["f32"], "m")
            close(d["v"].values(), v, 8 * EPS * (h[3] + h[1] ** 2) + TINY["f32"], "v")
            if "copy" in d:
                close(d["copy"].values(), got_p, rounding(got_p, "bf16"), "copy")
            h[0], h[2], h[3] = got_p, d["m"].values(), d["v"].values()


@pytest.mark.parametrize("gk", ["f32", "bf16"])
def test_adamw_8bit_states(gpu, gk):
    """From zeroed states; each step's states from the device's own last ones."""
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(32)
    tensors, host = [], []
    for i, n in enumerate([1, 2, 255, 256, 258, 4095, 4097, 9000]):
        off = i % 4
        nb = -(-n // 256)
        p, g = values(rng, (1, n), "f32"), values(rng, (1, n), gk, 1e-2)
        g[0, : n // 2] *= 2.0 ** -rng.integers(0, 30, n // 2)  # many sizes in a block
        g[0, n // 3] = 0.0
        if n > 600:
            g[0, 256:512] = 0.0  # a block of zeros
        d = dict(param=Mat(vs, st, p, "f32", off=off), grad=Mat(vs, st, g, gk, off=off),
                 m=Mat(vs, st, np.zeros((1, n)), "fp8", off=off),
                 v=Mat(vs, st, np.zeros((1, n)), "fp8", off=off),
                 m_scale=Mat(vs, st, np.zeros((1, nb)), "f32"),
                 v_scale=Mat(vs, st, np.zeros((1, nb)), "f32"),
                 copy=Mat(vs, st, None, "bf16", off=off, shape=(1, n)))
        tensors.append(d)
        host.append([p, unpack(pack(g, gk), gk), 0.05 * (i % 2)])
    print(f"adamw 8-bit states, {gk} gradients", flush=True)
    opt = vs.AdamW([dict({k: m.view for k, m in d.items()}, weight_decay=h[2])
                    for d, h in zip(tensors, host)], stream=st)

    def state(d):
        at = blocks_of(d["m"].cols)
        m = d["m"].values() * d["m_scale"].values()[:, at]
        r = d["v"].values() * d["v_scale"].values()[:, at]
        return m, r * r

    for step in (1, 2, 3):
        before = [state(d) for d in tensors]
        opt.step(step, stream=st, **HYPER)
        st.sync()
        for d, h, (m0, v0) in zip(tensors, host, before):
            n = d["m"].cols
            at = blocks_of(n)
            p, m, v = adamw_formula(h[0], h[1], m0, v0, h[2], step)
            move = np.abs(p - h[0]) + HYPER["lr"] * h[2] * np.abs(h[0])
            got = d["param"].values()
            close(got, p, 2 * EPS * (np.abs(p) + np.abs(h[0])) + 32 * EPS * move, "param")
            close(d["copy"].values(), got, rounding(got, "bf16"), "copy")
            for q, s, x in (("m", "m_scale", m), ("v", "v_scale", np.sqrt(v))):
                top = np.zeros(at[-1] + 1)
                np.maximum.at(top, at, np.abs(x[0]))
                scale = np.maximum(top, 1e-30) / 448
                close(d[s].values()[0], scale, 16 * EPS * scale, s)
                want = x / scale[at]
                # Half a step of e4m3, and a step below the smallest code for a
                # root that is kept off zero.
                tol = np.maximum(np.abs(want) * (2.0 ** -4 + 32 * EPS), 2.0 ** -10)
                if q == "v":
                    tol = np.where((want > 0) & (want < 2.0 ** -10), 2.0 ** -9, tol)
                    assert np.all(d["v"].values()[x > 1e-44] > 0)
                close(d[q].values(), want, tol, q)
            h[0] = got


def test_adamw_nan_stays_in_its_block(gpu):
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(33)
    n = 1024
    p, g = values(rng, (1, n), "f32"), values(rng, (1, n), "f32", 1e-2)
    g[0, 300] = np.nan
    d = dict(param=Mat(vs, st, p, "f32"), grad=Mat(vs, st, g, "f32"),
             m=Mat(vs, st, np.zeros((1, n)), "fp8"), v=Mat(vs, st, np.zeros((1, n)), "fp8"),
             m_scale=Mat(vs, st, np.zeros((1, 4)), "f32"),
             v_scale=Mat(vs, st, np.zeros((1, 4)), "f32"))
    vs.AdamW([{k: m.view for k, m in d.items()}], stream=st).step(1, stream=st, **HYPER)
    st.sync()
    bad = np.isnan(d["param"].values()[0])
    assert bad.sum() == 1 and bad[300]
    codes = np.isnan(d["m"].values()[0])
    assert codes[256:512].all() and not codes[:256].any() and not codes[512:].any()


# ------------------------------------------------------- streams, graphs, sizes
def test_empty_calls(gpu):
    """No rows: nothing is read or written, and sums over rows are zeros."""
    vs, st = gpu, gpu.Stream()
    w = vector(vs, st, np.ones(8))
    none = vs.DeviceView(0, (0, 8), vs.F32)
    vs.run_rmsnorm_gpu(none, w, none, stream=st)
    dw = vector(vs, st, np.full(8, 7.0))
    vs.run_rmsnorm_grad_gpu(none, none, w, vector(vs, st, [1.0]), none, dw, stream=st)
    W = Mat(vs, st, np.ones((5, 8)), "f32")
    DW = Mat(vs, st, np.ones((5, 8)), "f32", pad=3, off=1)
    out = vs.DeviceView(0, (0, 5), vs.F32)
    vs.run_linear_gpu(none, W.view, out, stream=st)
    db = vector(vs, st, np.full(5, 7.0))
    vs.run_linear_grad_gpu(out, none, W.view, dw=DW.view, dbias=db, stream=st)
    vs.AdamW([], stream=st).step(1, 1e-3, stream=st)
    st.sync()
    assert not dw.numpy(st).any() and not db.numpy(st).any() and not DW.values().any()


def test_rows_past_32_bit_offsets(gpu):
    """Rows spread over 9 GB: element offsets past 2^31, byte offsets past 2^32."""
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(40)
    M, C, ld = 2400, 64, 1 << 20
    big = vs.DeviceArray((M * ld,), np.float32)
    big.zero(st)
    rows = [0, 1, 1027, 2049, M - 2, M - 1]
    x = values(rng, (len(rows), C), "f32")
    for r, v in zip(rows, x.astype(np.float32)):
        vs._check(vs.load_library().vcsr_memcpy_h2d(big.ptr.value + 4 * r * ld, v.ctypes.data,
                                                    4 * C, st.h))
    view = vs.DeviceView(big.ptr, (M, C), vs.F32, ld=ld, owner=big)
    into = vs.DeviceView(big.ptr.value + 4 * 4096, (M, C), vs.F32, ld=ld, owner=big)
    w = np.ones(C)
    print("rows past 32-bit offsets: norm", flush=True)
    vs.run_rmsnorm_gpu(view, vector(vs, st, w), into, eps=1e-6, stream=st)
    wl = values(rng, (48, C), "f32")
    prod = vs.DeviceView(big.ptr.value + 4 * 8192, (M, 48), vs.F32, ld=ld, owner=big)
    print("rows past 32-bit offsets: linear", flush=True)
    vs.run_linear_gpu(view, Mat(vs, st, wl, "f32").view, prod, stream=st)
    dw = Mat(vs, st, None, "f32", shape=(48, C))
    print("rows past 32-bit offsets: linear grad", flush=True)
    vs.run_linear_grad_gpu(prod, view, Mat(vs, st, wl, "f32").view, dw=dw.view, stream=st)
    st.sync()

    def row(r, at, n):
        out = np.empty(n, np.float32)
        vs._check(vs.load_library().vcsr_memcpy_d2h(out.ctypes.data,
                                                    big.ptr.value + 4 * (r * ld + at), 4 * n, st.h))
        return out

    y = x @ wl.T
    for i, r in enumerate(rows):
        want = rms_norm(x[i:i + 1], None, w, 1e-6)[2][0]
        close(row(r, 4096, C), want, 40 * EPS * np.abs(want), f"norm row {r}")
        close(row(r, 8192, 48), y[i], 70 * EPS * (np.abs(x[i]) @ np.abs(wl).T), f"linear row {r}")
    assert not row(2048, 8192, 48).any()
    close(dw.values(), y.T @ x, 160 * EPS * (np.abs(y).T @ np.abs(x)), "dw")


def test_calls_repeat_bit_for_bit_and_replay_from_a_graph(gpu):
    """Every operator captured into one graph (kernel nodes alone), replayed
    between eager calls on new inputs: the same bits as the eager calls, which
    themselves repeat."""
    vs, st = gpu, gpu.Stream()
    hip = hip_runtime()
    rng = np.random.default_rng(50)
    M, K, N = 200, 520, 136
    lib = vs.load_library()

    def upload(mat, values_):
        host = mat.host.copy()
        mat.grid(host)[:, :mat.cols] = pack(values_, mat.kind)
        vs._check(lib.vcsr_memcpy_h2d(mat.buf.ptr, host.ctypes.data, host.nbytes, st.h))

    X, W = Mat(vs, st, None, "bf16", shape=(M, K)), Mat(vs, st, values(rng, (N, K), "bf16"), "bf16")
    U, S = Mat(vs, st, None, "bf16", shape=(M, K)), Mat(vs, st, None, "bf16", shape=(M, K))
    Y, Z = Mat(vs, st, None, "bf16", shape=(M, N)), Mat(vs, st, None, "bf16", shape=(M, N))
    DX, DU = Mat(vs, st, None, "bf16", shape=(M, K)), Mat(vs, st, None, "bf16", shape=(M, K))
    DW = Mat(vs, st, None, "bf16", shape=(N, K))
    nw, rstd = vector(vs, st, np.ones(K)), vector(vs, st, np.zeros(M))
    bias, db, dnw = (vector(vs, st, np.zeros(n)) for n in (N, N, K))
    P = Mat(vs, st, values(rng, (N, K), "f32"), "f32")
    m, v = (Mat(vs, st, np.zeros((N, K)), "fp8") for _ in range(2))
    ms, vsc = (vector(vs, st, np.zeros(-(-N * K // 256))) for _ in range(2))
    opt = vs.AdamW([dict(param=P.view, grad=DW.view, m=m.view, v=v.view, m_scale=ms, v_scale=vsc)],
                   stream=st)

    def step():
        vs.run_rmsnorm_gpu(X.view, nw, U.view, sum=S.view, rstd=rstd, stream=st)
        vs.run_linear_gpu(U.view, W.view, Y.view, bias=bias, act="gelu", z=Z.view, stream=st)
        vs.run_linear_grad_gpu(Y.view, U.view, W.view, z=Z.view, act="gelu", dx=DU.view,
                               dw=DW.view, dbias=db, stream=st)
        vs.run_rmsnorm_grad_gpu(DU.view, S.view, nw, rstd, DX.view, dnw, stream=st)
        opt.step(1, lr=1e-3, stream=st)

    start = [(b, b.numpy(st)) for b in (P.buf, m.buf, v.buf, ms, vsc)]

    def run(go, values_):
        upload(X, values_)
        for b, h in start:
            vs._check(lib.vcsr_memcpy_h2d(b.ptr, h.ctypes.data, h.nbytes, st.h))
        go()
        st.sync()
        return b"".join(b.numpy(st).tobytes() for b in
                        (Y.buf, Z.buf, DX.buf, DU.buf, DW.buf, db, dnw, P.buf, m.buf, v.buf, ms))

    inputs = [values(rng, (M, K), "bf16") for _ in range(3)]
    eager = [run(step, x) for x in inputs]
    assert eager[0] == run(step, inputs[0]) and eager[0] != eager[1]
    graph, kinds = capture(hip, st, step)
    gexec = ctypes.c_void_p()
    try:
        assert kinds and all(k == 0 for k in kinds), kinds
        assert hip.hipGraphInstantiateWithFlags(ctypes.byref(gexec), graph, 0) == 0

        def replay():
            assert hip.hipGraphLaunch(gexec, st.h) == 0

        for n in (0, 1, 2, 0):
            assert run(replay, inputs[n]) == eager[n], f"replay on input {n}"
            assert run(step, inputs[(n + 1) % 3]) == eager[(n + 1) % 3]
    finally:
        if gexec.value:
            hip.hipGraphExecDestroy(gexec)
        hip.hipGraphDestroy(graph)


def test_timed_calls_and_two_streams(gpu):
    """A timed call returns its time; calls on two streams with workspaces of
    their own do not disturb each other."""
    vs = gpu
    rng = np.random.default_rng(60)
    sts = [vs.Stream(), vs.Stream()]
    x, w = values(rng, (40, 6000), "f32"), values(rng, (300, 6000), "f32")
    outs = []
    for st in sts:
        X, W = Mat(vs, st, x, "f32"), Mat(vs, st, w, "f32")
        outs.append((st, X, W, Mat(vs, st, None, "f32", shape=(40, 300))))
    for _ in range(5):
        for st, X, W, Y in outs:
            vs.run_linear_gpu(X.view, W.view, Y.view, stream=st)
    for st in sts:
        st.sync()
    a, b = (o[3].codes().tobytes() for o in outs)
    assert a == b
    st, X, W, Y = outs[0]
    assert vs.run_linear_gpu(X.view, W.view, Y.view, stream=st, timed=True) > 0
    vs.release_workspaces()


def test_e4m3_table_is_the_devices(gpu):
    """Every code the norm can write, and its value: a row of e4m3's own values
    whose largest is 448 comes back code for code."""
    vs, st = gpu, gpu.Stream()
    codes = np.array([c for c in range(256) if c & 127 != 127], np.uint8)
    x = from_fp8(codes)[None, :]
    # rstd is a power of two for a mean square of one: scale the weight instead.
    t = np.where(codes & 128, -1.0, 1.0)[None, :]
    Y = Mat(vs, st, None, "fp8", shape=(1, len(codes)))
    scale = vector(vs, st, [0.0])
    vs.run_rmsnorm_gpu(Mat(vs, st, t, "f32").view, vector(vs, st, np.abs(x[0])), Y.view,
                       y_scale=scale, eps=0.0, stream=st)
    st.sync()
    assert scale.numpy(st)[0] == 1.0
    assert np.array_equal(E4M3[Y.codes()[0]], x[0])
