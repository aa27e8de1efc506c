"""The dense operators on the GPU where lifetimes, limits and shared buffers matter."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from conftest import capture, hip_runtime
from dense_ref import (EPS, Mat, act_grad, close, from_bf16, pack, rms_norm, rms_norm_grad, unpack,
                       vector)
from test_gpu_dense import check_norm, rounding, values

pytestmark = pytest.mark.gpu


def test_a_graph_outlives_the_workspace_it_was_captured_with(gpu):
    """A product whose sum is split, captured with the binding's workspace; then an eager
    call that needs a larger one, and buffers of the outgrown one's size: replays
    write none of them and give the eager call's bits."""
    vs, st = gpu, gpu.Stream()
    hip = hip_runtime()
    rng = np.random.default_rng(70)
    lib = vs.load_library()
    vs.release_workspaces()

    def product(M, N, K):
        x, w = rng.standard_normal((M, K)), rng.standard_normal((N, K)) / np.sqrt(K)
        X, W = Mat(vs, st, x, "f32"), Mat(vs, st, w, "f32")
        return X, W, Mat(vs, st, None, "f32", shape=(M, N)), x

    X, W, Y, x = product(64, 64, 8000)
    assert vs._linear_bytes(64, 64, 8000, 0, 0, False, False) > 0

    def step():
        vs.run_linear_gpu(X.view, W.view, Y.view, stream=st)

    step()
    st.sync()
    small = vs.workspace(1, st)
    graph, kinds = capture(hip, st, step)
    gexec = ctypes.c_void_p()
    try:
        assert kinds and all(k == 0 for k in kinds), kinds
        assert hip.hipGraphInstantiateWithFlags(ctypes.byref(gexec), graph, 0) == 0
        # A wide gradient: dz alone is larger than the first workspace.
        M, N, K = 3000, 512, 64
        dy, z, xx = (Mat(vs, st, rng.standard_normal((M, n)), "f32") for n in (N, N, K))
        ww, dx = Mat(vs, st, rng.standard_normal((N, K)), "f32"), \
            Mat(vs, st, None, "f32", shape=(M, K))
        vs.run_linear_grad_gpu(dy.view, xx.view, ww.view, z=z.view, act="silu", dx=dx.view,
                               stream=st)
        st.sync()
        large = vs.workspace(1, st)
        assert large is not small and large.nbytes > small.nbytes
        guards = [vs.DeviceArray.from_numpy(np.full(small.nbytes, 0x5B, np.uint8), st)
                  for _ in range(3)]
        for n in range(3):
            values = x * (n + 1)
            host = X.host.copy()
            X.grid(host)[:, :X.cols] = pack(values, "f32")
            vs._check(lib.vcsr_memcpy_h2d(X.buf.ptr, host.ctypes.data, host.nbytes, st.h))
            step()
            st.sync()
            eager = Y.codes().tobytes()
            Y.buf.copy_from(vs.DeviceArray.from_numpy(Y.host, st), st)
            st.sync()
            print(f"replay {n}", flush=True)
            assert hip.hipGraphLaunch(gexec, st.h) == 0
            st.sync()
            assert np.array_equal(Y.codes().view(np.uint8).ravel(), np.frombuffer(eager, np.uint8))
            assert all((g.numpy(st) == 0x5B).all() for g in guards)
    finally:
        if gexec.value:
            hip.hipGraphExecDestroy(gexec)
        hip.hipGraphDestroy(graph)
    vs.release_workspaces()


def put(vs, st, array, at, values_):
    """values_ to element `at` of a device array."""
    v = np.ascontiguousarray(values_, array.dtype)
    vs._check(vs.load_library().vcsr_memcpy_h2d(array.ptr.value + at * v.itemsize, v.ctypes.data,
                                                v.nbytes, st.h))


def take(vs, st, array, at, n):
    out = np.empty(n, array.dtype)
    vs._check(vs.load_library().vcsr_memcpy_d2h(out.ctypes.data,
                                                array.ptr.value + at * out.itemsize, out.nbytes,
                                                st.h))
    return out


@pytest.mark.parametrize("kinds, C", [("f32 f32", 3), ("f32 fp8", 1), ("bf16 bf16", 7),
                                      ("bf16 fp8", 2), ("bf16 f32", 5)])
def test_rmsnorm_of_millions_of_narrow_rows(gpu, kinds, C):
    """Rows shorter than a vector, more of them than 2^32 threads would be at 1024 a row."""
    xk, yk = kinds.split()
    rng = np.random.default_rng(C)
    M = (1 << 22) + 3
    print(f"narrow rows {kinds} {M}x{C}", flush=True)
    x, r = values(rng, (M, C), xk), values(rng, (M, C), xk)
    w = (1 + 0.2 * rng.standard_normal(C)).astype(np.float32).astype(np.float64)
    check_norm(gpu, gpu.Stream(), x, r, w, xk, yk, 1e-6, f"{kinds} {M}x{C}", pad=C % 2, off=1)


@pytest.mark.parametrize("kinds, C", [("f32 f32", 3), ("bf16 bf16", 7), ("f32 bf16", 2)])
@pytest.mark.parametrize("M", [1, 255, 257, 5000, (1 << 22) + 3])
def test_rmsnorm_grad_of_narrow_rows(gpu, kinds, C, M):
    xk, yk = kinds.split()
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(M % 1000 + C)
    print(f"narrow rows grad {kinds} {M}x{C}", flush=True)
    s, dy = values(rng, (M, C), xk, 1.5), values(rng, (M, C), yk)
    ds = values(rng, (M, C), xk)
    w = (1 + 0.2 * rng.standard_normal(C)).astype(np.float32).astype(np.float64)
    rstd = (1 / np.sqrt(np.mean(s * s, axis=1) + 1e-6)).astype(np.float32)
    DX = Mat(vs, st, None, xk, 1, 1, (M, C))
    dweight = vector(vs, st, np.full(C, np.nan))
    vs.run_rmsnorm_grad_gpu(Mat(vs, st, dy, yk, 2, 1).view, Mat(vs, st, s, xk, 0, 1).view,
                            vector(vs, st, w), vector(vs, st, rstd), DX.view, dweight,
                            dsum=Mat(vs, st, ds, xk).view, stream=st)
    st.sync()
    rd = rstd.astype(np.float64)[:, None]
    want, want_w = rms_norm_grad(dy, s, w, rd, ds)
    h, g = np.abs(s * rd), np.abs(dy * w)
    dot = np.sum(g * h, axis=1, keepdims=True) / C
    tol = 8 * EPS * (rd * (g + h * dot) + np.abs(want)) + rd * h * dot * (C + 4) * EPS
    close(DX.values(), want, tol + rounding(want, xk), "dx")
    # A thread's chain of at most 17 rows, 6 steps over lanes, 3 over waves, and the
    # partial rows: 16 a thread, then 14; 3 roundings in each product.
    close(dweight.numpy(st), want_w, 64 * EPS * np.sum(np.abs(dy) * h, axis=0) + 1e-30, "dweight")


def test_rmsnorm_of_rows_for_two_launches(gpu):
    """64 threads a row and 2^26 rows: in place, 35 GB."""
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(80)
    M, C = (1 << 26) + 5, 132
    big = vs.DeviceArray((M, C), np.float32)
    big.zero(st)
    rstd = vs.DeviceArray((M,), np.float32)
    rstd.zero(st)
    rows = [0, 1, (1 << 26) - 257, (1 << 26) - 256, (1 << 26) - 1, 1 << 26, M - 1]
    x = rng.standard_normal((len(rows), C)).astype(np.float32)
    w = (1 + 0.2 * rng.standard_normal(C)).astype(np.float32)
    for r, v in zip(rows, x):
        put(vs, st, big, r * C, v)
    print("rows for two launches", flush=True)
    vs.run_rmsnorm_gpu(big, vector(vs, st, w), big, rstd=rstd, eps=1e-6, stream=st)
    st.sync()
    u = (C / 8 + 16) * EPS
    for r, v in zip(rows, x.astype(np.float64)):
        _, want_r, want = rms_norm(v[None], None, w.astype(np.float64), 1e-6)
        close(take(vs, st, big, r * C, C), want[0], np.abs(want[0]) * (u + 5 * EPS), f"row {r}")
        close(take(vs, st, rstd, r, 1), want_r[0], want_r[0] * u, f"rstd {r}")
    zero = take(vs, st, rstd, (1 << 26) - 255, 3)
    close(zero, np.full(3, 1e3), np.full(3, 1e3) * u, "rstd of zeros")
    assert not take(vs, st, big, 12345678 * C, C).any()


def test_rmsnorm_grad_of_columns_for_two_launches(gpu):
    """64 threads add up a column of dweight's partial rows: 2^26 columns."""
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(81)
    M, C = 2, (1 << 26) + 5
    s, dy, dx = (vs.DeviceArray((M, C), np.float32) for _ in range(3))
    w, dweight = vs.DeviceArray((C,), np.float32), vs.DeviceArray((C,), np.float32)
    for a in (s, dy, w):
        a.zero(st)
    rstd = np.float32([0.5, 2.0])
    cols = [0, 31, (1 << 25) - 1, 1 << 25, (1 << 26) - 1, 1 << 26, C - 1]
    sv, dv = rng.standard_normal((M, len(cols))), rng.standard_normal((M, len(cols)))
    for m in range(M):
        for i, c in enumerate(cols):
            put(vs, st, s, m * C + c, np.float32([sv[m, i]]))
            put(vs, st, dy, m * C + c, np.float32([dv[m, i]]))
    put(vs, st, dweight, 0, np.full(C, 7, np.float32))
    print("columns for two launches", flush=True)
    vs.run_rmsnorm_grad_gpu(dy, s, w, vector(vs, st, rstd), dx, dweight, stream=st)
    st.sync()
    got = dweight.numpy(st)
    sv, dv = sv.astype(np.float32).astype(np.float64), dv.astype(np.float32).astype(np.float64)
    terms = dv * sv * rstd[:, None]
    close(got[cols], terms.sum(0), 4 * EPS * np.abs(terms).sum(0), "dweight")
    got[cols] = 0
    assert not got.any()
    vs.release_workspaces()


def test_no_rows_and_a_large_weight_gradient(gpu):
    """Zeros in 17 GB of dw, and in a million rows with a gap between them, by a kernel each."""
    vs, st = gpu, gpu.Stream()
    N, K = 1 << 17, (1 << 15) + 8
    big = vs.DeviceArray((N, K), np.float32)
    vs._check(vs.load_library().vcsr_memset_d(big.ptr, 0x5B, big.nbytes, st.h))
    x, dy = vs.DeviceView(0, (0, K), vs.F32), vs.DeviceView(0, (0, N), vs.F32)
    w = vs.DeviceView(big.ptr, (N, K), vs.F32)
    print("17 GB of zeros", flush=True)
    vs.run_linear_grad_gpu(dy, x, w, dw=big, stream=st)
    st.sync()
    for at in (0, 1 << 30, (1 << 32) - 4, 1 << 32, N * K - 64):
        assert not take(vs, st, big, at, 64).any(), at
    N = 1 << 20  # the most outputs of a gradient
    DW = Mat(vs, st, np.ones((N, 1)), "bf16", pad=2, off=1)
    db = vector(vs, st, np.ones(N))
    print("rows with gaps", flush=True)
    vs.run_linear_grad_gpu(vs.DeviceView(0, (0, N), vs.F32), vs.DeviceView(0, (0, 1), vs.BF16),
                           DW.view, dw=DW.view, dbias=db, stream=st)
    st.sync()
    assert not DW.codes().any() and not db.numpy(st).any()


def test_linear_of_more_rows_than_small_tiles_have_blocks(gpu):
    """2^30 + 3 rows: 64 x 64 tiles of 256 threads would need 2^32 threads."""
    vs, st = gpu, gpu.Stream()
    M = (1 << 30) + 3
    x, y = vs.DeviceArray((M, 1), np.float32), vs.DeviceArray((M, 1), np.float32)
    x.zero(st)
    vs._check(vs.load_library().vcsr_memset_d(y.ptr, 0x5B, y.nbytes, st.h))
    rows = [0, 63, (1 << 29) + 1, (1 << 30) - 1, 1 << 30, M - 1]
    for r in rows:
        put(vs, st, x, r, np.float32([r % 1000 + 0.5]))
    print("2^30 rows", flush=True)
    vs.run_linear_gpu(x, vector(vs, st, [[3.0]]), y, bias=vector(vs, st, [-1.0]), stream=st)
    st.sync()
    for r in rows:
        assert take(vs, st, y, r, 1)[0] == 3 * (r % 1000 + 0.5) - 1, r
    assert (take(vs, st, y, 1 << 28, 1000) == -1).all()
    assert (take(vs, st, y, M - 100, 96) == -1).all()


@pytest.mark.parametrize("C", [3, 100, 2000, 20000])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_rmsnorm_grad_in_place(gpu, kind, C):
    """dx over dsum, s and dy: the bits of dx and dweight apart."""
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(C)
    M = 70
    host = {k: values(rng, (M, C), kind) for k in ("dy", "s", "dsum")}
    w = vector(vs, st, 1 + 0.1 * rng.standard_normal(C))
    rstd = vector(vs, st, 0.5 + rng.random(M))
    want = None
    for over in (None, "dsum", "s", "dy"):
        mats = {k: Mat(vs, st, v, kind, pad=8) for k, v in host.items()}
        dx = mats[over] if over else Mat(vs, st, None, kind, pad=8, shape=(M, C))
        dweight = vector(vs, st, np.full(C, np.nan))
        print(f"norm gradient in place {kind} C={C} over {over}", flush=True)
        vs.run_rmsnorm_grad_gpu(mats["dy"].view, mats["s"].view, w, rstd, dx.view, dweight,
                                dsum=mats["dsum"].view, stream=st)
        st.sync()
        got = (dx.codes().tobytes(), dweight.numpy(st).tobytes())
        want = want or got
        same = got == want  # no difference of megabytes in the message
        assert same, over


@pytest.mark.parametrize("out, over", [("y", "x"), ("y", "w"), ("z", "x"), ("z", "w")])
def test_linear_refuses_outputs_over_operands(gpu, out, over):
    """Refused before any launch: nothing is written."""
    vs, st = gpu, gpu.Stream()
    n = 40
    mats = {k: Mat(vs, st, np.full((n, n), i + 1.0), "f32") for i, k in enumerate("xwyz")}
    kw = {k: m.view for k, m in mats.items()}
    kw[out] = kw[over]
    with pytest.raises(vs.VcsrError) as e:
        vs.run_linear_gpu(stream=st, **kw)
    assert e.value.code == vs.VCSR_EINVAL and f"{out}: another matrix" in str(e.value)
    st.sync()
    for i, k in enumerate("xwyz"):
        assert (mats[k].values() == i + 1).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_linear_grad_over_what_no_product_reads(gpu, kind):
    """dx over x without dw, over dy and z with an activation; dw over w without dx:
    the bits of a call apart."""
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(90)
    n = 200
    host = {k: values(rng, (n, n), kind) for k in ("dy", "x", "w", "z")}

    def call(out, over):
        m = {k: Mat(vs, st, v, kind) for k, v in host.items()}
        to = m[over] if over else Mat(vs, st, None, kind, shape=(n, n))
        vs.run_linear_grad_gpu(m["dy"].view, m["x"].view, m["w"].view, z=m["z"].view, act="silu",
                               stream=st, **{out: to.view})
        st.sync()
        return to.codes().tobytes()

    for out, over in (("dx", "x"), ("dx", "dy"), ("dx", "z"), ("dw", "w"), ("dw", "dy")):
        print(f"{out} over {over} {kind}", flush=True)
        same = call(out, over) == call(out, None)
        assert same, (out, over)


@pytest.mark.parametrize("act", ["relu", "gelu", "silu"])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_activation_gradients_of_every_magnitude(gpu, kind, act):
    """act'(z) over the whole range of z, a column each (dbias of one row of ones):
    a finite z has a finite gradient, also where z^2 or z^3 is past FP32's range."""
    vs, st = gpu, gpu.Stream()
    if kind == "bf16":
        z = from_bf16(np.arange(1 << 16, dtype=np.uint16))
        z = z[np.isfinite(z)].astype(np.float64)
    else:
        z = np.concatenate([np.linspace(-30, 30, 4001), 2.0 ** np.linspace(-126, 127.9, 3000),
                            -2.0 ** np.linspace(-126, 127.9, 3000)])
    z = unpack(pack(z[None, :], kind), kind)
    n = z.shape[1]
    one = np.ones((1, n))
    db = vector(vs, st, np.full(n, np.nan))
    print(f"act' {act} {kind}", flush=True)
    vs.run_linear_grad_gpu(Mat(vs, st, one, kind).view, Mat(vs, st, np.ones((1, 1)), kind).view,
                           Mat(vs, st, one.T, kind).view, z=Mat(vs, st, z, kind).view, act=act,
                           dbias=db, stream=st)
    st.sync()
    z = z[0]
    # act' = p + b p (1 - p) for p = 1 / (1 + e^-u).  The sum and the reciprocal round p
    # (4 u of it), the exponential's argument u and itself move it by p (1 - p) (|u| + 2)
    # 4 u; where e^-u is under 2^-26, p is one and what it lacks is lost.  1e-30: p
    # past FP32's range.
    with np.errstate(all="ignore"):
        k = 2 * np.sqrt(2 / np.pi)
        arg, b = (k * (z + 0.044715 * z ** 3), np.abs(z) * k * (1 + 0.134145 * z * z)) \
            if act == "gelu" else (z, np.abs(z))
        p, q = 1 / (1 + np.exp(-arg)), 1 / (1 + np.exp(arg))
        # Not through tanh, whose 1 + t and 1 - t^2 lose what is small.
        want = act_grad(z, act) if act == "relu" else p + np.sign(z) * b * p * q
        dp = np.where(np.exp(-arg) < 2.0 ** -26, q, 4 * EPS * p + 4 * EPS * p * q * (np.abs(arg) + 2))
        tol = dp + np.where(dp > 0, dp * b, 0) + np.where(q > 0, 8 * EPS * p * q * b, 0)
    tol = np.zeros(n) if act == "relu" else np.nan_to_num(tol) + 4 * EPS * np.abs(want) + 1e-30
    assert np.isfinite(want).all() and tol.max() < 2.0 ** -16
    close(db.numpy(st), want, tol, f"{act} {kind}")


@pytest.mark.parametrize("kinds", ["f32 fp8", "bf16 fp8"])
@pytest.mark.parametrize("C", [2, 40, 130, 700, 6001, 20000])
def test_rmsnorm_scales_where_x_times_weight_leaves_the_range(gpu, kinds, C):
    """|x w| under and over FP32's range where y = x / rms(x) w is not."""
    xk, yk = kinds.split()
    rng = np.random.default_rng(C)
    st = gpu.Stream()
    for size, gain in ((2.0 ** -60, 2.0 ** -90), (2.0 ** 50, 2.0 ** 82), (2.0 ** -60, 2.0 ** 60),
                       (2.0 ** 50, 2.0 ** -80)):
        print(f"scales {kinds} C={C} x {size:g} weight {gain:g}", flush=True)
        x = values(rng, (5, C), xk, size)
        x[1] *= 2.0 ** 3
        w = (gain * (1 + 0.2 * rng.standard_normal(C))).astype(np.float32).astype(np.float64)
        check_norm(gpu, st, x, None, w, xk, yk, 0.0, f"{kinds} {C}", with_sum=False)
