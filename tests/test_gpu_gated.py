"""The gated projection and its gradients on the GPU against the formulas in 64 bits;
the tolerances are block_ref's."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from block_ref import gated, gated_grad, rounding, values
from conftest import capture, hip_runtime
from dense_plans import STEP, TILES
from dense_ref import EPS, Mat, act, act_grad, close, pack, unpack, vector
from gated_plans import forced, gated_grad_plan, gated_plan
from test_gpu_dense_kernels import FORWARD, sums

pytestmark = pytest.mark.gpu


def gated_once(vs, st, rng, M, N, K, xk, yk, kind, pad=0, off=0, bias="gu", with_z=False):
    """Weights of two strides; x, weights and outputs at odd addresses for an odd `off`."""
    x = values(rng, (M, K), xk)
    wg, wu = values(rng, (N, K), xk, K ** -0.5), values(rng, (N, K), xk, K ** -0.5)
    scales = [None] * 3
    if xk == "fp8":
        scales = [(0.5 + rng.random(n)).astype(np.float32) for n in (M, N, N)]
    b = [(0.3 * rng.standard_normal(N)).astype(np.float32) if k in bias else None for k in "gu"]
    X, G = Mat(vs, st, x, xk, pad, off), Mat(vs, st, wg, xk, pad, off)
    U = Mat(vs, st, wu, xk, 2 * pad, 3 * off)
    Y = Mat(vs, st, None, yk, pad, off, (M, N))
    Z = [Mat(vs, st, None, yk, pad, off, (M, N)) for _ in range(2)] if with_z else [None] * 2

    def dev(v):
        return None if v is None else vector(vs, st, v)

    vs.run_gated_gpu(X.view, G.view, U.view, Y.view, gate_bias=dev(b[0]), up_bias=dev(b[1]),
                     act=kind, z_gate=Z[0].view if with_z else None,
                     z_up=Z[1].view if with_z else None, x_scale=dev(scales[0]),
                     gate_scale=dev(scales[1]), up_scale=dev(scales[2]), stream=st)
    st.sync()
    x, wg, wu = (v if s is None else v * s.astype(np.float64)[:, None]
                 for v, s in zip((x, wg, wu), scales))
    b = [None if v is None else v.astype(np.float64) for v in b]
    want, tol = gated(x, wg, wu, *b, kind)
    what = f"{M}x{N}x{K} {xk} {yk} {kind}"
    for mat, v, t, name in zip((*Z, Y), want, tol, ("z_gate", "z_up", "y")):
        if mat:
            close(mat.values(), v, t + rounding(v, yk), f"{name} {what}")
    return Y.codes()


def grad_once(vs, st, rng, M, N, K, xk, yk, kind, pad=0, off=0, want=("dx", "dw", "g", "u")):
    x = values(rng, (M, K), xk)
    wg, wu = values(rng, (N, K), xk, K ** -0.5), values(rng, (N, K), xk, K ** -0.5)
    zg, zu, dy = (values(rng, (M, N), yk) for _ in range(3))
    X, G, U = (Mat(vs, st, v, xk, p, off) for v, p in ((x, pad), (wg, pad), (wu, 2 * pad)))
    ZG, ZU = Mat(vs, st, zg, yk, pad, off), Mat(vs, st, zu, yk, pad, 2 * off)
    DY = Mat(vs, st, dy, yk, 3 * pad, off)
    DX, DG = Mat(vs, st, None, xk, pad, off, (M, K)), Mat(vs, st, None, xk, pad, off, (N, K))
    DU = Mat(vs, st, None, xk, 2 * pad, 3 * off, (N, K))
    bg, bu = (vector(vs, st, np.full(N, np.nan)) for _ in range(2))
    vs.run_gated_grad_gpu(DY.view, X.view, G.view, U.view, ZG.view, ZU.view, act=kind,
                          dx=DX.view if "dx" in want else None,
                          dw_gate=DG.view if "dw" in want else None,
                          dw_up=DU.view if "dw" in want else None,
                          dgate_bias=bg if "g" in want else None,
                          dup_bias=bu if "u" in want else None, stream=st)
    st.sync()
    (dx, dg, du, vg, vu), (tx, tg, tu, tbg, tbu) = gated_grad(dy, x, wg, wu, zg, zu, kind, xk)
    what = f"{M}x{N}x{K} {xk} {yk} {kind}"
    if "dx" in want:
        close(DX.values(), dx, tx + rounding(dx, xk), "dx " + what)
    if "dw" in want:
        close(DG.values(), dg, tg + rounding(dg, xk), "dw_gate " + what)
        close(DU.values(), du, tu + rounding(du, xk), "dw_up " + what)
    if "g" in want:
        close(bg.numpy(st), vg, tbg, "dgate_bias " + what)
    if "u" in want:
        close(bu.numpy(st), vu, tbu, "dup_bias " + what)


SHAPES = [(1, 1, 1), (1, 64, 64), (3, 5, 7), (8, 33, 65), (17, 129, 40), (64, 64, 128),
          (65, 31, 130), (129, 200, 257), (300, 47, 514), (1, 1000, 4100), (9, 260, 2051),
          (130, 300, 1030)]
TYPES = ["f32 f32", "f32 bf16", "bf16 bf16", "bf16 f32", "fp8 bf16", "fp8 f32"]


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_gated(gpu, shape, types):
    xk, yk = types.split()
    st, rng = gpu.Stream(), np.random.default_rng(sum(shape))
    for n, (kind, pad, off, bias) in enumerate((("gelu", 0, 0, "gu"), ("silu", 1, 1, "g"),
                                                ("relu", 16, 0, "u"), ("none", 8, 3, ""))):
        print(f"gated {types} {shape} {kind} pad={pad} off={off}", flush=True)
        gated_once(gpu, st, rng, *shape, xk, yk, kind, pad, off, bias, with_z=n % 2 == 0)


@pytest.mark.parametrize("types", ["f32 f32", "bf16 bf16", "fp8 bf16"])
@pytest.mark.parametrize("shape", [(2048, 1024, 192), (4099, 515, 96), (700, 2048, 640),
                                   (2500, 500, 72), (513, 4100, 256), (7956, 1024, 1024),
                                   (5001, 2048, 512)], ids=lambda s: "x".join(map(str, s)))
def test_gated_many_tiles(gpu, shape, types):
    """Sizes that fill the chip, whole and ragged."""
    xk, yk = types.split()
    print(f"gated {types} {shape}", flush=True)
    gated_once(gpu, gpu.Stream(), np.random.default_rng(3), *shape, xk, yk, "silu", with_z=True)


@pytest.mark.parametrize("kind, tile, stages", FORWARD)
def test_gated_kernels(gpu, kind, tile, stages):
    st, rng = gpu.Stream(), np.random.default_rng(tile + stages)
    yk = "f32" if kind == "f32" else "bf16"
    for n, K in enumerate(sums(kind)):
        for M, N, pad, off in ((1, 1, 0, 0), (255, 129, 0, 0), (257, 150, 3, 1), (300, 127, 16, 0)):
            print(f"gated {kind} {tile}/{stages} {M}x{N}x{K} pad={pad} off={off}", flush=True)
            with forced(gpu, tile, stages):
                gated_once(gpu, st, rng, M, N, K, kind, yk, ("gelu", "silu", "relu", "none")[n % 4],
                           pad, off, bias="gu" if n % 2 else "", with_z=n % 3 == 0)


@pytest.mark.parametrize("kind, tile, stages", FORWARD)
def test_gated_kernels_with_split_sums(gpu, kind, tile, stages):
    """Two and three parts (added a thread each) and nine and more (by eight), the last
    one shorter, of one step and of none that is whole."""
    st, rng = gpu.Stream(), np.random.default_rng(tile + stages + 1)
    s = STEP[kind]
    for splits, K in ((2, 3 * s), (2, 2 * s + 1), (3, 5 * s - 1), (9, 9 * s), (12, 23 * s + 5)):
        for M, N, pad, off in ((1, 7, 0, 0), (257, 150, 0, 0), (130, 123, 5, 1)):
            print(f"gated {kind} {tile}/{stages} {M}x{N}x{K} in {splits}", flush=True)
            with forced(gpu, tile, stages, splits):
                gated_once(gpu, st, rng, M, N, K, kind, "f32", "silu", pad, off, with_z=True)


@pytest.mark.parametrize("kind, tile, stages", FORWARD)
def test_gated_kernels_with_divided_rows(gpu, kind, tile, stages):
    st, rng = gpu.Stream(), np.random.default_rng(tile + stages + 2)
    for M, rows in ((2 * tile, tile), (2 * tile + 1, 2 * tile), (3 * tile - 1, tile)):
        print(f"gated {kind} {tile}/{stages} {rows} of {M} rows", flush=True)
        with forced(gpu, tile, stages, rows=rows):
            gated_once(gpu, st, rng, M, 130, 2 * STEP[kind] + 9, kind, "bf16", "gelu", 3, 1,
                       with_z=True)


@pytest.mark.parametrize("kind", list(TILES))
def test_gated_rows_kernel(gpu, kind):
    """Up to 16 rows: sums of one to three turns of a wave's 8 lines of 128 bytes, whole
    and ragged."""
    st, rng = gpu.Stream(), np.random.default_rng(16)
    line = STEP[kind]
    for K in (1, line - 1, 16 * line, 17 * line + 1, 32 * line, 33 * line, 64 * line,
              64 * line + 1, 65 * line, 129 * line - 3):
        for M, N, pad, off in ((1, 150, 0, 0), (7, 17, 0, 0), (8, 9, 16, 0), (16, 33, 3, 1)):
            print(f"gated rows {kind} {M}x{N}x{K} pad={pad} off={off}", flush=True)
            with forced(gpu, 16):
                gated_once(gpu, st, rng, M, N, K, kind, "bf16", "silu", pad, off, with_z=M == 8)


GATED_SIZES = [  # M, N, K, type -> tile, stages, splits, rows
    (2, 1050, 9000, "bf16", (16, 1, 1, 2)),
    (64, 500, 4100, "bf16", (64, 4, None, 64)),
    (7956, 1024, 1000, "bf16", (256, 2, 1, 7956)),
    (7956, 1024, 1016, "fp8", (256, 2, 1, 7956)),
    (5001, 2048, 700, "bf16", (256, 2, 1, 4096)),
    (5001, 2048, 500, "f32", (128, 2, 1, 4096)),
]


@pytest.mark.parametrize("size", GATED_SIZES, ids=lambda s: "x".join(map(str, s[:4])))
def test_gated_sizes_choose_their_kernels(gpu, size):
    M, N, K, kind, want = size
    got = gated_plan(gpu, M, N, K, kind)
    assert all(w is None or g == w for g, w in zip(got, want)), got
    print(f"gated {M}x{N}x{K} {kind}", flush=True)
    gated_once(gpu, gpu.Stream(), np.random.default_rng(7), M, N, K, kind, "bf16", "gelu")


def test_gated_keeps_nan_and_infinity_in_their_rows(gpu):
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(4)
    for kind in ("f32", "bf16"):
        for M, N, K in ((5, 40, 100), (200, 150, 70)):
            x = values(rng, (M, K), kind)
            wg, wu = (unpack(pack(np.abs(rng.standard_normal((N, K))) + 0.5, kind), kind)
                      for _ in range(2))
            x[1, K - 1], x[2, 0] = np.nan, np.inf
            Y = Mat(vs, st, None, "f32", shape=(M, N))
            vs.run_gated_gpu(*(Mat(vs, st, v, kind).view for v in (x, wg, wu)), Y.view, act="relu",
                             stream=st)
            st.sync()
            y = Y.values()
            assert np.isnan(y[1]).all() and (y[2] == np.inf).all()
            assert np.isfinite(np.delete(y, (1, 2), 0)).all()


def test_gated_weights_that_are_one_matrix(gpu):
    """Both weights in one buffer, one behind the other and row by row in turn: the bits
    of two."""
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(11)
    M, N, K = 70, 90, 100
    x, w = values(rng, (M, K), "bf16"), values(rng, (2, N, K), "bf16")
    X = Mat(vs, st, x, "bf16")
    got = []
    for layout in ("two", "behind", "turn"):
        if layout == "two":
            G, U = (Mat(vs, st, v, "bf16").view for v in w)
        elif layout == "behind":
            both = Mat(vs, st, w.reshape(2 * N, K), "bf16")
            G, U = (vs.DeviceView(both.buf.ptr.value + h * N * K * 2, (N, K), vs.BF16, owner=both)
                    for h in (0, 1))
        else:
            both = Mat(vs, st, w.transpose(1, 0, 2).reshape(2 * N, K), "bf16")
            G, U = (vs.DeviceView(both.buf.ptr.value + h * K * 2, (N, K), vs.BF16, ld=2 * K,
                                  owner=both) for h in (0, 1))
        Y = Mat(vs, st, None, "f32", shape=(M, N))
        vs.run_gated_gpu(X.view, G, U, Y.view, stream=st)
        st.sync()
        got.append(Y.codes().tobytes())
    assert got[0] == got[1] == got[2]


# ------------------------------------------------------------------ gradients
@pytest.mark.parametrize("types", ["f32 f32", "bf16 bf16", "bf16 f32", "f32 bf16"])
@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 64, 96), (3, 5, 7), (33, 65, 31), (64, 128, 64),
                                   (100, 130, 70), (500, 47, 260), (2100, 40, 136),
                                   (1000, 300, 520)], ids=lambda s: "x".join(map(str, s)))
def test_gated_grad(gpu, shape, types):
    xk, yk = types.split()
    st, rng = gpu.Stream(), np.random.default_rng(sum(shape))
    for kind, pad, off in (("gelu", 0, 0), ("silu", 8, 0), ("relu", 3, 1), ("none", 0, 0)):
        print(f"gated grad {types} {shape} {kind} pad={pad} off={off}", flush=True)
        grad_once(gpu, st, rng, *shape, xk, yk, kind, pad, off)
    for want in (("dx",), ("dw",), ("g",), ("u",), ("dx", "g"), ("dw", "u"), ("dx", "dw")):
        print(f"gated grad {types} {shape} {want}", flush=True)
        grad_once(gpu, st, rng, *shape, xk, yk, "silu", want=want)


GRAD = [(k, t) for k in ("f32", "bf16") for t, s in TILES[k] if s == 2]


@pytest.mark.parametrize("together", [False, True], ids=["apart", "together"])
@pytest.mark.parametrize("kind, tile", GRAD)
def test_gated_gradient_kernels(gpu, kind, tile, together):
    """dw sums over the rows, dx over the outputs of both weights, whole steps and ends
    of each, in parts that begin and end in either."""
    st, rng = gpu.Stream(), np.random.default_rng(tile)
    s = sums(kind)
    for n, (M, N, K) in enumerate([(1, 1, 1), (s[1], s[3], 257), (s[2], 255, 300),
                                   (s[3], s[4], 300), (s[4], 300, 1), (s[5], s[5], 257),
                                   (300, s[6], 255), (257, s[2], 300), (s[6], 520, 264)]):
        for splits in (1, 3):
            pad, off = ((0, 0), (8, 0), (3, 1))[(n + splits) % 3]
            print(f"gated gradient {kind} {tile} {M}x{N}x{K} in {splits} pad={pad}", flush=True)
            with forced(gpu, tile, 2, splits, together=together):
                grad_once(gpu, st, rng, M, N, K, kind, kind, ("gelu", "relu", "none")[n % 3], pad,
                          off)
        if not together:
            for splits in (2, 5):
                with forced(gpu, tile, 2, splits):
                    for want in (("dx",), ("dw", "g", "u")):
                        print(f"gated gradient {kind} {tile} {M}x{N}x{K} {want}", flush=True)
                        grad_once(gpu, st, rng, M, N, K, kind, kind, "silu", want=want)


@pytest.mark.parametrize("tile", [64, 128, 256])
def test_gated_gradient_kernels_with_many_parts(gpu, tile):
    st, rng = gpu.Stream(), np.random.default_rng(tile + 3)
    for kind in ("f32", "bf16"):
        if tile == 256 and kind == "f32":
            continue
        for splits, together in ((9, True), (20, False)):
            print(f"gated gradient {kind} {tile} in {splits} together={together}", flush=True)
            with forced(gpu, tile, 2, splits, together=together):
                grad_once(gpu, st, rng, 20 * STEP[kind] + 1, 136, 260, kind, kind, "gelu")


GRAD_SIZES = [  # M, N, K, type
    (8192, 2048, 1024, "bf16"), (2000, 2000, 1500, "bf16"), (2000, 2000, 1500, "f32"),
    (4100, 264, 2200, "bf16"), (3000, 2500, 64, "f32"),
]


@pytest.mark.parametrize("size", GRAD_SIZES, ids=lambda s: "x".join(map(str, s[:4])))
def test_gated_gradient_sizes(gpu, size):
    M, N, K, kind = size
    print(f"gated gradient {M}x{N}x{K} {kind}", gated_grad_plan(gpu, M, N, K, kind), flush=True)
    grad_once(gpu, gpu.Stream(), np.random.default_rng(8), M, N, K, kind, kind, "gelu")


# Few rows: dx's long sum is split, dw is whole, and both are one launch.
FEW_ROWS = [(1, 2752, 64, "bf16"), (9, 1551, 384, "f32"), (10, 603, 1780, "f32"),
            (84, 6272, 64, "bf16"), (239, 1536, 64, "f32")]


@pytest.mark.parametrize("size", FEW_ROWS, ids=lambda s: "x".join(map(str, s)))
def test_gated_gradient_of_few_rows(gpu, size):
    M, N, K, kind = size
    together, tile_w, splits_w, tile_x, splits_x = gated_grad_plan(gpu, M, N, K, kind)
    assert together and tile_w == tile_x and splits_w == 1 and splits_x > 1
    grad_once(gpu, gpu.Stream(), np.random.default_rng(23), M, N, K, kind, kind, "gelu")


def test_gated_grad_against_differences(gpu):
    """The directional derivative of <dy, y> along a random direction of all inputs."""
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(19)
    M, N, K = 6, 20, 24
    for kind in ("gelu", "silu", "none"):
        x, wg, wu = values(rng, (M, K), "f32"), values(rng, (N, K), "f32"), values(rng, (N, K), "f32")
        bg, bu = values(rng, (1, N), "f32"), values(rng, (1, N), "f32")
        dy = values(rng, (M, N), "f32")
        d = [rng.standard_normal(v.shape) for v in (x, wg, wu, bg, bu)]

        def loss(t):
            a, g, u, p, q = (v + t * e for v, e in zip((x, wg, wu, bg, bu), d))
            return np.sum(dy * act(a @ g.T + p, kind) * (a @ u.T + q))

        h = 1e-5
        diff = (loss(h) - loss(-h)) / (2 * h)
        mats = [Mat(vs, st, v, "f32") for v in (x, wg, wu)]
        Y, ZG, ZU = (Mat(vs, st, None, "f32", shape=(M, N)) for _ in range(3))
        vs.run_gated_gpu(*(m.view for m in mats), Y.view, gate_bias=vector(vs, st, bg[0]),
                         up_bias=vector(vs, st, bu[0]), act=kind, z_gate=ZG.view, z_up=ZU.view,
                         stream=st)
        DX, DG, DU = Mat(vs, st, None, "f32", shape=(M, K)), Mat(vs, st, None, "f32", shape=(N, K)), \
            Mat(vs, st, None, "f32", shape=(N, K))
        db = [vector(vs, st, np.zeros(N)) for _ in range(2)]
        vs.run_gated_grad_gpu(Mat(vs, st, dy, "f32").view, *(m.view for m in mats), ZG.view,
                              ZU.view, act=kind, dx=DX.view, dw_gate=DG.view, dw_up=DU.view,
                              dgate_bias=db[0], dup_bias=db[1], stream=st)
        st.sync()
        got = [DX.values(), DG.values(), DU.values(), *(v.numpy(st)[None] for v in db)]
        parts = [g * e for g, e in zip(got, d)]
        size = sum(np.sum(np.abs(p)) for p in parts)
        # Differences are good to h^2 and 2^-52 / h; the gradients to 2^-18 of their terms
        # (sums of 24 products, their error through act' and both factors).
        assert abs(diff - sum(np.sum(p) for p in parts)) <= (2.0 ** -18 + 1e-8) * size, kind


def test_gated_of_no_rows(gpu):
    vs, st = gpu, gpu.Stream()
    N, K = 40, 70
    W = [Mat(vs, st, np.ones((N, K)), "bf16", 3, 1) for _ in range(2)]
    x, y = vs.DeviceView(0, (0, K), vs.BF16), vs.DeviceView(0, (0, N), vs.F32)
    vs.run_gated_gpu(x, W[0].view, W[1].view, y, stream=st)
    D = [Mat(vs, st, np.ones((N, K)), "bf16", 2, 1) for _ in range(2)]
    b = [vector(vs, st, np.ones(N)) for _ in range(2)]
    vs.run_gated_grad_gpu(y, x, W[0].view, W[1].view, y, y, dx=x, dw_gate=D[0].view,
                          dw_up=D[1].view, dgate_bias=b[0], dup_bias=b[1], stream=st)
    st.sync()
    assert not any(m.values().any() for m in D) and not any(v.numpy(st).any() for v in b)


@pytest.mark.parametrize("M, kind", [(3, "bf16"), (300, "bf16"), (130, "f32")])
def test_gated_replayed_from_a_graph(gpu, M, kind):
    """Projection and gradient captured, replayed between eager calls on other rows."""
    vs, st = gpu, gpu.Stream()
    hip, lib = hip_runtime(), vs.load_library()
    rng = np.random.default_rng(12)
    N, K = 200, 1030
    x = values(rng, (M, K), kind)
    X, DY = Mat(vs, st, x, kind), Mat(vs, st, values(rng, (M, N), kind), kind)
    W = [Mat(vs, st, values(rng, (N, K), kind, K ** -0.5), kind) for _ in range(2)]
    Y, ZG, ZU = (Mat(vs, st, None, kind, shape=(M, N)) for _ in range(3))
    DX, DG, DU = Mat(vs, st, None, kind, shape=(M, K)), Mat(vs, st, None, kind, shape=(N, K)), \
        Mat(vs, st, None, kind, shape=(N, K))
    b = [vector(vs, st, np.zeros(N)) for _ in range(2)]

    def step():
        vs.run_gated_gpu(X.view, W[0].view, W[1].view, Y.view, z_gate=ZG.view, z_up=ZU.view,
                         stream=st)
        vs.run_gated_grad_gpu(DY.view, X.view, W[0].view, W[1].view, ZG.view, ZU.view, dx=DX.view,
                              dw_gate=DG.view, dw_up=DU.view, dgate_bias=b[0], dup_bias=b[1],
                              stream=st)

    outs = (Y, ZG, ZU, DX, DG, DU)

    def bits():
        st.sync()
        return tuple(m.codes().tobytes() for m in outs) + tuple(v.numpy(st).tobytes() for v in b)

    step()
    graph, kinds = capture(hip, st, step)
    gexec = ctypes.c_void_p()
    try:
        assert kinds and all(k == 0 for k in kinds), kinds  # kernels only
        assert hip.hipGraphInstantiateWithFlags(ctypes.byref(gexec), graph, 0) == 0
        for n in range(3):
            host = X.host.copy()
            X.grid(host)[:, :K] = pack(x * (n + 1) / 2, kind)
            vs._check(lib.vcsr_memcpy_h2d(X.buf.ptr, host.ctypes.data, host.nbytes, st.h))
            step()
            eager = bits()
            for m in outs:
                m.buf.copy_from(vs.DeviceArray.from_numpy(m.host, st), st)
            for v in b:
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


def test_gated_grad_over_what_no_product_reads(gpu):
    """dx over x without dw, over dy and z (which are read before); dw over the weights
    without dx: the bits of a call apart."""
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(90)
    n = 200
    for kind in ("f32", "bf16"):
        host = {k: values(rng, (n, n), kind) for k in ("dy", "x", "w_gate", "w_up", "z_gate", "z_up")}

        def call(out, over):
            m = {k: Mat(vs, st, v, kind) for k, v in host.items()}
            to = [m[o] if o else Mat(vs, st, None, kind, shape=(n, n)) for o in over]
            vs.run_gated_grad_gpu(**{k: v.view for k, v in m.items()}, stream=st,
                                  **{k: v.view for k, v in zip(out, to)})
            st.sync()
            return [v.codes().tobytes() for v in to]

        dw = ("dw_gate", "dw_up")
        for out, over in ((("dx",), ("x",)), (("dx",), ("dy",)), (("dx",), ("z_gate",)),
                          (("dx",), ("z_up",)), (dw, ("w_gate", "w_up")), (dw, ("z_up", "dy"))):
            print(f"{out} over {over} {kind}", flush=True)
            same = call(out, over) == call(out, [None] * len(out))
            assert same, (out, over)


@pytest.mark.parametrize("kind", ["relu", "gelu", "silu", "none"])
def test_gated_grad_formula_by_elements(gpu, kind):
    """One row, one weight column of ones each: dbias are the two dz, at every z."""
    vs, st = gpu, gpu.Stream()
    z = np.concatenate([np.linspace(-30, 30, 4001), 2.0 ** np.linspace(-60, 20, 500),
                        -2.0 ** np.linspace(-60, 20, 500)]).astype(np.float32).astype(np.float64)[None]
    n = z.shape[1]
    zu, dy = np.full((1, n), 3.0), np.full((1, n), -0.5)
    b = [vector(vs, st, np.full(n, np.nan)) for _ in range(2)]
    one = Mat(vs, st, np.ones((n, 1)), "f32").view
    vs.run_gated_grad_gpu(Mat(vs, st, dy, "f32").view, Mat(vs, st, np.ones((1, 1)), "f32").view, one,
                          one, Mat(vs, st, z, "f32").view, Mat(vs, st, zu, "f32").view, act=kind,
                          dgate_bias=b[0], dup_bias=b[1], stream=st)
    st.sync()
    with np.errstate(all="ignore"):
        want = act(z[0], kind)
        slope = act_grad(z[0], kind)
    close(b[1].numpy(st), -0.5 * want, 10 * EPS * np.abs(z[0]) + 1e-30, f"dz_up {kind}")
    close(b[0].numpy(st), -1.5 * slope, 1.5 * 40 * EPS * 1.13 + 0 * z[0], f"dz_gate {kind}")
