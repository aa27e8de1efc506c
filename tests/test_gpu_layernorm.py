"""Layer norm and its gradient on the GPU against the formulas in 64 bits; the
tolerances are block_ref's."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from block_ref import layer_norm, layer_norm_grad, layer_norm_tol, rounding, values
from conftest import capture, hip_runtime
from dense_ref import EPS, Mat, close, pack, unpack, vector

pytestmark = pytest.mark.gpu


def gain(rng, C):
    return (1 + 0.2 * rng.standard_normal(C)).astype(np.float32).astype(np.float64)


def shift(rng, C):
    return (0.3 * rng.standard_normal(C)).astype(np.float32).astype(np.float64)


def check(vs, st, x, r, w, b, xk, yk, eps, what, pad=0, off=0, with_sum=True):
    M, C = x.shape
    X = Mat(vs, st, x, xk, pad, off)
    R = Mat(vs, st, r, xk, pad, 2 * off) if r is not None else None
    S = Mat(vs, st, None, xk, pad, off, (M, C)) if with_sum else None
    Y = Mat(vs, st, None, yk, pad, off, (M, C))
    scale = vector(vs, st, np.zeros(M)) if yk == "fp8" else None
    mean, rstd = vector(vs, st, np.zeros(M)), vector(vs, st, np.zeros(M))
    vs.run_layernorm_gpu(X.view, vector(vs, st, w), Y.view,
                         bias=vector(vs, st, b) if b is not None else None,
                         residual=R.view if R else None, sum=S.view if S else None, y_scale=scale,
                         mean=mean, rstd=rstd, eps=eps, stream=st)
    st.sync()
    X.codes()
    eps = float(np.float32(eps))
    with np.errstate(all="ignore"):
        t, m, rs, want = layer_norm(x, r, w, b, eps)
        tm, tr, ty = layer_norm_tol(t, m, rs, w, b, eps)
    fine = np.isfinite(want).all(axis=1, keepdims=True)
    want = np.where(fine, want, np.nan)  # all of such a row
    tm, tr, ty = (np.where(fine, v, 0) for v in (tm, tr, ty))
    rows = fine[:, 0]
    close(mean.numpy(st)[rows], m[rows, 0], tm[rows, 0], what + " mean")
    close(rstd.numpy(st)[rows], rs[rows, 0], tr[rows, 0], what + " rstd")
    if S:
        close(S.values(), t, EPS * np.abs(t) + rounding(t, xk), what + " sum")
    if yk != "fp8":
        close(Y.values(), want, ty + rounding(np.nan_to_num(want), yk), what)
        return Y
    top, worst = np.max(np.abs(want), axis=1), np.max(ty, axis=1)
    want_scale = np.where(top < 1e-30, 1e-30, top) / 448
    close(scale.numpy(st), want_scale, np.nan_to_num(worst / 448 + 4 * EPS * want_scale),
          what + " scale")
    q = want / want_scale[:, None]
    e = np.nan_to_num(ty / want_scale[:, None] + np.abs(q) * (worst / 448 / want_scale + 8 * EPS)[:, None])
    close(Y.values(), q, e + np.maximum((np.abs(np.nan_to_num(q)) + e) * 2.0 ** -4, 2.0 ** -10), what)
    return Y


KINDS = ["f32 f32", "f32 bf16", "f32 fp8", "bf16 f32", "bf16 bf16", "bf16 fp8"]


@pytest.mark.parametrize("C", [1, 3, 8, 31, 64, 128, 130, 257, 512, 1000, 2050, 4096, 8191, 9001,
                               17001])
@pytest.mark.parametrize("kinds", KINDS)
def test_layernorm(gpu, kinds, C):
    xk, yk = kinds.split()
    st, rng = gpu.Stream(), np.random.default_rng(C)
    for M, pad, off, residual, bias in ((1, 0, 0, True, True), (5, 3, 1, True, False),
                                        (67, 0, 0, False, True)):
        print(f"layernorm {kinds} C={C} M={M} pad={pad} off={off}", flush=True)
        x = values(rng, (M, C), xk, 2.0)
        r = values(rng, (M, C), xk) if residual else None
        check(gpu, st, x, r, gain(rng, C), shift(rng, C) if bias else None, xk, yk, 1e-5,
              f"{kinds} {M}x{C}", pad=pad, off=off)


@pytest.mark.parametrize("kinds", ["f32 f32", "bf16 fp8"])
@pytest.mark.parametrize("C", [5, 64, 700, 3000, 12000, 20000])
def test_layernorm_of_rows_far_from_zero(gpu, kinds, C):
    """Means 256 times the deviation: a sum of squares alone would lose the variance."""
    xk, yk = kinds.split()
    st, rng = gpu.Stream(), np.random.default_rng(C)
    print(f"layernorm far {kinds} C={C}", flush=True)
    x = rng.standard_normal((6, C)) + 256 * np.sign(rng.standard_normal((6, 1)))
    check(gpu, st, unpack(pack(x, xk), xk), None, gain(rng, C), shift(rng, C), xk, yk,
          1e-5, f"{kinds} far {C}")


@pytest.mark.parametrize("kinds", ["f32 f32", "bf16 bf16", "bf16 fp8", "f32 fp8"])
@pytest.mark.parametrize("C", [3, 32, 512, 8192, 32768])
def test_layernorm_rows_that_are_constant_or_not_finite(gpu, kinds, C):
    """Rows of zeros, of one value (whose sum is exact), tiny and huge ones, and rows
    with a NaN or an infinity, which reach no other row."""
    xk, yk = kinds.split()
    st, rng = gpu.Stream(), np.random.default_rng(C)
    x = values(rng, (9, C), xk)
    x[1], x[2] = 0, -2.5
    x[3] *= 2.0 ** -60
    x[4] *= 2.0 ** 40
    x[5, C // 2], x[6, C - 1], x[7, 0] = np.nan, np.inf, -np.inf
    w = gain(rng, C)
    w[C // 3] = 0
    print(f"layernorm edge rows {kinds} C={C}", flush=True)
    check(gpu, st, x, None, w, shift(rng, C), xk, yk, 1e-5, f"{kinds} edge rows", with_sum=False)
    check(gpu, st, x[:5], None, w, None, xk, yk, 1e-12, f"{kinds} edge rows", with_sum=False)


def test_layernorm_past_the_range_of_its_sums(gpu):
    """Squares past FP32: rstd 0 and y the bias; a sum past it: NaN, in its row alone."""
    vs, st = gpu, gpu.Stream()
    for C in (7, 200, 9000):
        x = np.zeros((3, C))
        x[0, :2] = 1e25, -1e25
        x[1] = 3e38
        x[2, 1] = 1
        w, b = np.full(C, 2.0), np.arange(C) % 7 - 3.0
        Y, rstd = Mat(vs, st, None, "f32", shape=(3, C)), vector(vs, st, np.ones(3))
        vs.run_layernorm_gpu(Mat(vs, st, x, "f32").view, vector(vs, st, w), Y.view,
                             bias=vector(vs, st, b), rstd=rstd, stream=st)
        st.sync()
        y = Y.values()
        assert rstd.numpy(st)[0] == 0 and np.array_equal(y[0], b)
        assert np.isnan(y[1]).all() and np.isfinite(y[2]).all()


def test_layernorm_in_place(gpu):
    """sum over x and over the residual, y over x and over the residual: the same bits
    as apart."""
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(5)
    for kind in ("f32", "bf16"):
        for C in (3, 100, 2000, 2050, 20000):
            print(f"layernorm in place {kind} C={C}", flush=True)
            x, r = values(rng, (70, C), kind), values(rng, (70, C), kind)
            w, b = vector(vs, st, gain(rng, C)), vector(vs, st, shift(rng, C))

            def call(sum_over, y_over):
                m = {"x": Mat(vs, st, x, kind), "residual": Mat(vs, st, r, kind)}
                S = m.get(sum_over) or Mat(vs, st, None, kind, shape=(70, C))
                Y = m.get(y_over) or Mat(vs, st, None, kind, shape=(70, C))
                vs.run_layernorm_gpu(m["x"].view, w, Y.view, bias=b, residual=m["residual"].view,
                                     sum=S.view, stream=st)
                st.sync()
                return S.codes().tobytes(), Y.codes().tobytes()

            apart = call(None, None)
            for over in (("x", None), ("residual", None), (None, "x"), (None, "residual"),
                         ("x", "residual"), ("residual", "x")):
                same = call(*over) == apart
                assert same, over


GRAD_KINDS = ["f32 f32", "bf16 bf16", "f32 bf16", "bf16 f32"]


def check_grad(vs, st, rng, M, C, xk, yk, pad=0, off=0, dsum=True, scale=1.5):
    s, dy = values(rng, (M, C), xk, scale), values(rng, (M, C), yk)
    s = s + 2.0 if xk == "f32" else s
    ds = values(rng, (M, C), xk) if dsum else None
    w = gain(rng, C)
    _, mean, rstd, _ = layer_norm(s, None, w, None, 1e-5)
    mean, rstd = mean[:, 0].astype(np.float32), rstd[:, 0].astype(np.float32)
    S, DY = Mat(vs, st, s, xk, pad, off), Mat(vs, st, dy, yk, pad, 2 * off)
    DS = Mat(vs, st, ds, xk, pad, off) if dsum else None
    DX = Mat(vs, st, None, xk, pad, off, (M, C))
    dweight, dbias = vector(vs, st, np.full(C, np.nan)), vector(vs, st, np.full(C, np.nan))
    vs.run_layernorm_grad_gpu(DY.view, S.view, vector(vs, st, w), vector(vs, st, mean),
                              vector(vs, st, rstd), DX.view, dweight, dbias,
                              dsum=DS.view if DS else None, stream=st)
    st.sync()
    # s as the kernel has it: 2 added to FP32 values rounds once.
    s = S.values()
    (dx, dw, db), (tx, tw, tb) = layer_norm_grad(dy, s, w, mean.astype(np.float64)[:, None],
                                                 rstd.astype(np.float64)[:, None], ds)
    what = f"{xk} {yk} {M}x{C}"
    close(DX.values(), dx, tx + rounding(dx, xk), f"dx {what}")
    close(dweight.numpy(st), dw, tw, f"dweight {what}")
    close(dbias.numpy(st), db, tb, f"dbias {what}")


@pytest.mark.parametrize("C", [1, 7, 64, 130, 600, 2050, 8191, 9001, 17001])
@pytest.mark.parametrize("kinds", GRAD_KINDS)
def test_layernorm_grad(gpu, kinds, C):
    xk, yk = kinds.split()
    st, rng = gpu.Stream(), np.random.default_rng(100 + C)
    for M, pad, off, dsum in ((1, 0, 0, True), (6, 5, 1, False), (1500, 0, 0, True)):
        if M * C > 4e6:
            M = 300
        print(f"layernorm grad {kinds} C={C} M={M}", flush=True)
        check_grad(gpu, st, rng, M, C, xk, yk, pad, off, dsum)


# Vectors of 16 bytes a row: one for each choice of waves and vectors a lane, at its
# ends, and the first length that is read more than once.
VECTORS = [1, 2, 3, 64, 65, 128, 129, 192, 193, 256, 257, 384, 385, 512, 513, 768, 769, 1024, 1025,
           1536, 1537, 2048, 2049]


@pytest.mark.parametrize("vectors", VECTORS)
@pytest.mark.parametrize("kinds", ["f32 bf16", "bf16 fp8"])
def test_layernorm_rows_of_every_shape(gpu, kinds, vectors):
    xk, yk = kinds.split()
    V = 4 if xk == "f32" else 8
    rng, st = np.random.default_rng(vectors), gpu.Stream()
    for C in (vectors * V, vectors * V - V + 1, vectors * V - 1):
        if C < V:
            continue
        for M, pad, off in ((3, 0, 0), (9, 5, 1)):
            print(f"layernorm {kinds} {M}x{C}", flush=True)
            check(gpu, st, values(rng, (M, C), xk), values(rng, (M, C), xk), gain(rng, C),
                  shift(rng, C), xk, yk, 1e-5, f"{kinds} {M}x{C}", pad=pad, off=off)


@pytest.mark.parametrize("vectors", VECTORS)
@pytest.mark.parametrize("kinds", ["f32 bf16", "bf16 f32"])
def test_layernorm_gradient_rows_of_every_shape(gpu, kinds, vectors):
    xk, yk = kinds.split()
    V = 4 if xk == "f32" else 8
    rng, st = np.random.default_rng(vectors), gpu.Stream()
    for C, M in ((vectors * V, 5), (vectors * V - 1, 5), (vectors * V - V + 1, 300)):
        if C < V:
            continue
        print(f"layernorm gradient {kinds} {M}x{C}", flush=True)
        check_grad(gpu, st, rng, M, C, xk, yk, 3, 1)


@pytest.mark.parametrize("kinds, C", [("f32 f32", 3), ("f32 fp8", 1), ("bf16 bf16", 7),
                                      ("bf16 f32", 64)])
def test_layernorm_of_many_rows(gpu, kinds, C):
    """Rows that a row group takes in turn, and more of them than its blocks."""
    xk, yk = kinds.split()
    rng, M = np.random.default_rng(C), (1 << 20) + 3
    print(f"layernorm {kinds} {M}x{C}", flush=True)
    check(gpu, gpu.Stream(), values(rng, (M, C), xk), values(rng, (M, C), xk), gain(rng, C),
          shift(rng, C), xk, yk, 1e-5, f"{kinds} {M}x{C}", pad=C % 2, off=1)


@pytest.mark.parametrize("C", [3, 100, 2000, 20000])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_layernorm_grad_in_place(gpu, kind, C):
    """dx over dsum, s and dy: the bits of dx, dweight and dbias apart; and those of
    calls that ask for one of the two sums."""
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(C)
    M = 1100
    host = {k: values(rng, (M, C), kind) for k in ("dy", "s", "dsum")}
    w, mean = vector(vs, st, gain(rng, C)), vector(vs, st, 0.1 * rng.standard_normal(M))
    rstd = vector(vs, st, 0.5 + rng.random(M))

    def call(over, sums="wb"):
        mats = {k: Mat(vs, st, v, kind, pad=8) for k, v in host.items()}
        dx = mats[over] if over else Mat(vs, st, None, kind, pad=8, shape=(M, C))
        dw, db = (vector(vs, st, np.full(C, np.nan)) if k in sums else None for k in "wb")
        print(f"layernorm gradient {kind} C={C} over {over} {sums}", flush=True)
        vs.run_layernorm_grad_gpu(mats["dy"].view, mats["s"].view, w, mean, rstd, dx.view, dw, db,
                                  dsum=mats["dsum"].view, stream=st)
        st.sync()
        return (dx.codes().tobytes(), *(v.numpy(st).tobytes() if v else None for v in (dw, db)))

    want = call(None)
    for over in ("dsum", "s", "dy"):
        same = call(over) == want  # no difference of megabytes in the message
        assert same, over
    for sums in ("w", "b", ""):
        got = call(None, sums)
        assert all(g is None or g == v for g, v in zip(got, want)), sums


def test_layernorm_grad_against_differences(gpu):
    """The directional derivative of <dy, y> along a random direction, by central
    differences of the formula, against the kernel's gradients."""
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(9)
    M, C = 5, 96
    x, dy = values(rng, (M, C), "f32"), values(rng, (M, C), "f32")
    w, b = gain(rng, C), shift(rng, C)
    _, mean, rstd, _ = layer_norm(x, None, w, b, 1e-5)
    DX = Mat(vs, st, None, "f32", shape=(M, C))
    dweight, dbias = vector(vs, st, np.zeros(C)), vector(vs, st, np.zeros(C))
    vs.run_layernorm_grad_gpu(Mat(vs, st, dy, "f32").view, Mat(vs, st, x, "f32").view,
                              vector(vs, st, w), vector(vs, st, mean[:, 0]),
                              vector(vs, st, rstd[:, 0]), DX.view, dweight, dbias, stream=st)
    st.sync()
    vx, vw, vb, h = rng.standard_normal((M, C)), rng.standard_normal(C), rng.standard_normal(C), 1e-5

    def loss(t):
        return np.sum(dy * layer_norm(x + t * vx, None, w + t * vw, b + t * vb, 1e-5)[3])

    diff = (loss(h) - loss(-h)) / (2 * h)
    parts = (DX.values() * vx, dweight.numpy(st).astype(np.float64) * vw,
             dbias.numpy(st).astype(np.float64) * vb)
    # Differences are good to h^2 and 2^-52 / h; the gradients to 2^-20 of their terms.
    size = sum(np.sum(np.abs(p)) for p in parts)
    assert abs(diff - sum(np.sum(p) for p in parts)) <= (2.0 ** -20 + 1e-8) * size


def test_layernorm_of_no_rows(gpu):
    """Nothing is written but zeros in the sums."""
    vs, st = gpu, gpu.Stream()
    x = vs.DeviceView(0, (0, 40), vs.F32)
    w = vector(vs, st, np.ones(40))
    vs.run_layernorm_gpu(x, w, x, bias=w, stream=st)
    dw, db = vector(vs, st, np.ones(40)), vector(vs, st, np.ones(40))
    none = vs.DeviceView(0, (0,), vs.F32)
    vs.run_layernorm_grad_gpu(x, x, w, none, none, x, dw, db, stream=st)
    st.sync()
    assert not dw.numpy(st).any() and not db.numpy(st).any()


def test_layernorm_past_4_gib(gpu):
    """Byte offsets past 2^32: rows at both ends of 9 GB, in place."""
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(3)
    M, C = 70000, 32769
    big = vs.DeviceArray((M, C), np.float32)
    big.zero(st)
    lib, rows = vs.load_library(), [0, 1, 32767, 32768, 65535, M - 1]
    x = rng.standard_normal((len(rows), C)).astype(np.float32)
    for r, v in zip(rows, x):
        vs._check(lib.vcsr_memcpy_h2d(big.ptr.value + r * C * 4, v.ctypes.data, v.nbytes, st.h))
    w, b = gain(rng, C), shift(rng, C)
    vs.run_layernorm_gpu(big, vector(vs, st, w), big, bias=vector(vs, st, b), stream=st)
    st.sync()
    x = x.astype(np.float64)
    _, mean, rstd, y = layer_norm(x, None, w, b, float(np.float32(1e-5)))
    tol = layer_norm_tol(x, mean, rstd, w, b, 1e-5)[2]
    got = np.empty(C, np.float32)
    for i, r in enumerate(rows):
        vs._check(lib.vcsr_memcpy_d2h(got.ctypes.data, big.ptr.value + r * C * 4, got.nbytes, st.h))
        close(got, y[i], tol[i] + EPS * np.abs(y[i]), f"row {r}")
    vs._check(lib.vcsr_memcpy_d2h(got.ctypes.data, big.ptr.value + 50000 * C * 4, got.nbytes, st.h))
    assert np.array_equal(got, b.astype(np.float32))


def test_layernorm_replayed_from_a_graph(gpu):
    """Forward and gradient captured, replayed between eager calls on new values."""
    vs, st = gpu, gpu.Stream()
    hip, lib = hip_runtime(), vs.load_library()
    rng = np.random.default_rng(12)
    M, C = 900, 520
    x, dy = values(rng, (M, C), "bf16"), values(rng, (M, C), "bf16")
    X, DY = Mat(vs, st, x, "bf16"), Mat(vs, st, dy, "bf16")
    Y, DX = Mat(vs, st, None, "fp8", shape=(M, C)), Mat(vs, st, None, "bf16", shape=(M, C))
    w, b = vector(vs, st, gain(rng, C)), vector(vs, st, shift(rng, C))
    scale, mean, rstd = (vector(vs, st, np.zeros(M)) for _ in range(3))
    dw, db = vector(vs, st, np.zeros(C)), vector(vs, st, np.zeros(C))

    def step():
        vs.run_layernorm_gpu(X.view, w, Y.view, bias=b, y_scale=scale, mean=mean, rstd=rstd,
                             stream=st)
        vs.run_layernorm_grad_gpu(DY.view, X.view, w, mean, rstd, DX.view, dw, db, stream=st)

    def bits():
        st.sync()
        return (Y.codes().tobytes(), DX.codes().tobytes(),
                *(v.numpy(st).tobytes() for v in (scale, mean, rstd, dw, db)))

    step()
    graph, kinds = capture(hip, st, step)
    gexec = ctypes.c_void_p()
    try:
        assert kinds and all(k == 0 for k in kinds), kinds  # kernels only
        assert hip.hipGraphInstantiateWithFlags(ctypes.byref(gexec), graph, 0) == 0
        for n in range(3):
            host = X.host.copy()
            X.grid(host)[:, :C] = pack(x * (n + 1) + n, "bf16")
            vs._check(lib.vcsr_memcpy_h2d(X.buf.ptr, host.ctypes.data, host.nbytes, st.h))
            step()
            eager = bits()
            for m in (Y, DX):
                m.buf.copy_from(vs.DeviceArray.from_numpy(m.host, st), st)
            for v in (scale, mean, rstd, dw, db):
                v.zero(st)
            st.sync()
            print(f"replay {n}", flush=True)
            assert hip.hipGraphLaunch(gexec, st.h) == 0
            same = bits() == eager
            assert same, n
    finally:
        if gexec.value:
            hip.hipGraphExecDestroy(gexec)
        hip.hipGraphDestroy(graph)
