"""Every kernel of the dense products at small odd sizes, the sizes that choose the
large ones by themselves, and every row shape of the norm."""
from __future__ import annotations

import numpy as np
import pytest

from dense_plans import STEP, TILES, forced, grad_plan, linear_plan
from dense_ref import EPS, Mat, close, rms_norm_grad, vector
from test_gpu_dense import check_norm, grad_once, linear_once, rounding, values

pytestmark = pytest.mark.gpu

FORWARD = [(k, *t) for k in TILES for t in TILES[k]]
GRAD = [(k, t) for k in ("f32", "bf16") for t, s in TILES[k] if s == 2]


def sums(kind):
    """Lengths of a sum around whole steps, odd numbers of steps among them."""
    s = STEP[kind]
    return [1, s - 1, s, s + 1, 2 * s + 3, 3 * s, 5 * s - 2]


@pytest.mark.parametrize("kind, tile, stages", FORWARD)
def test_forward_kernels(gpu, kind, tile, stages):
    st, rng = gpu.Stream(), np.random.default_rng(tile + stages)
    yk = "f32" if kind == "f32" else "bf16"
    for n, K in enumerate(sums(kind)):
        for M, N, pad, off in ((1, 1, 0, 0), (255, 257, 0, 0), (257, 300, 3, 1), (300, 255, 16, 0)):
            print(f"{kind} {tile}/{stages} {M}x{N}x{K} pad={pad} off={off}", flush=True)
            with forced(gpu, tile, stages):
                linear_once(gpu, st, rng, M, N, K, kind, yk, ("gelu", "silu", "relu", "none")[n % 4],
                            pad, off, residual=n % 2 == 0, with_z=n % 3 == 0)


@pytest.mark.parametrize("kind, tile, stages", FORWARD)
def test_forward_kernels_with_split_sums(gpu, kind, tile, stages):
    """Two and three parts (added a thread each) and nine and more (by eight), the last
    one shorter, of one step and of none that is whole."""
    st, rng = gpu.Stream(), np.random.default_rng(tile + stages + 1)
    s = STEP[kind]
    for splits, K in ((2, 3 * s), (2, 2 * s + 1), (3, 5 * s - 1), (9, 9 * s), (12, 23 * s + 5)):
        for M, N, pad, off in ((1, 7, 0, 0), (257, 300, 0, 0), (130, 255, 5, 1)):
            print(f"{kind} {tile}/{stages} {M}x{N}x{K} in {splits}", flush=True)
            with forced(gpu, tile, stages, splits):
                linear_once(gpu, st, rng, M, N, K, kind, "f32", "silu", pad, off, with_z=True)


@pytest.mark.parametrize("kind, tile, stages", FORWARD)
def test_forward_kernels_with_divided_rows(gpu, kind, tile, stages):
    st, rng = gpu.Stream(), np.random.default_rng(tile + stages + 2)
    for M, rows in ((2 * tile, tile), (2 * tile + 1, 2 * tile), (3 * tile - 1, tile)):
        print(f"{kind} {tile}/{stages} {rows} of {M} rows", flush=True)
        with forced(gpu, tile, stages, rows=rows):
            linear_once(gpu, st, rng, M, 260, 2 * STEP[kind] + 9, kind, "bf16", "gelu", 3, 1,
                        with_z=True)


@pytest.mark.parametrize("kind", list(TILES))
def test_rows_kernel(gpu, kind):
    """Up to 16 rows: sums of one to three turns of a wave's 8 lines of 128 bytes, whole
    and ragged."""
    st, rng = gpu.Stream(), np.random.default_rng(16)
    line = STEP[kind]
    for K in (1, line - 1, 16 * line, 17 * line + 1, 32 * line, 33 * line, 64 * line,
              64 * line + 1, 65 * line, 128 * line, 129 * line - 3):
        for M, N, pad, off in ((1, 300, 0, 0), (7, 17, 0, 0), (8, 33, 16, 0), (16, 65, 3, 1)):
            print(f"rows {kind} {M}x{N}x{K} pad={pad} off={off}", flush=True)
            with forced(gpu, 16):
                linear_once(gpu, st, rng, M, N, K, kind, "bf16", "silu", pad, off, with_z=M == 8)


@pytest.mark.parametrize("together", [False, True], ids=["apart", "together"])
@pytest.mark.parametrize("kind, tile", GRAD)
def test_gradient_kernels(gpu, kind, tile, together):
    """dw sums over the rows, dx over the outputs; a dx or dw that is alone has its
    kernel to itself."""
    st, rng = gpu.Stream(), np.random.default_rng(tile)
    s = sums(kind)
    for n, (M, N, K) in enumerate([(1, 1, 1), (s[1], s[3], 257), (s[2], 255, 300),
                                   (s[3], s[4], 300), (s[4], 300, 1), (s[5], s[5], 257),
                                   (300, s[6], 255), (257, s[2], 300), (s[6], 520, 264)]):
        for splits in (1, 3):
            pad, off = ((0, 0), (8, 0), (3, 1))[(n + splits) % 3]
            print(f"gradient {kind} {tile} {M}x{N}x{K} in {splits} pad={pad}", flush=True)
            with forced(gpu, tile, 2, splits, together=together):
                grad_once(gpu, st, rng, M, N, K, kind, kind, ("gelu", "relu", "none")[n % 3], pad,
                          off)
        if not together:
            with forced(gpu, tile, 2, 2):
                for want in (("dx",), ("dw", "dbias")):
                    grad_once(gpu, st, rng, M, N, K, kind, kind, "silu", want=want)


@pytest.mark.parametrize("tile", [64, 128, 256])
def test_gradient_kernels_with_many_parts(gpu, tile):
    """dw over many rows in 9 and 20 parts, dbias' partial rows in the same launch."""
    st, rng = gpu.Stream(), np.random.default_rng(tile + 3)
    for kind in ("f32", "bf16"):
        if tile == 256 and kind == "f32":
            continue
        for splits, together in ((9, True), (20, False)):
            print(f"gradient {kind} {tile} in {splits} together={together}", flush=True)
            with forced(gpu, tile, 2, splits, together=together):
                grad_once(gpu, st, rng, 20 * STEP[kind] + 1, 136, 260, kind, kind, "gelu")


# ------------------------------------------------ sizes and the kernels they are for
LINEAR_SIZES = [  # M, N, K, type -> tile, stages, splits, rows
    (2, 2100, 9000, "bf16", (16, 1, 1, 2)),
    (8, 2048, 2500, "f32", (16, 1, 1, 8)),
    (64, 1000, 4100, "bf16", (64, 4, None, 64)),
    (2500, 1000, 72, "fp8", (64, 2, 1, 2500)),
    (7956, 2048, 1000, "bf16", (256, 2, 1, 7956)),
    (7956, 2048, 1016, "fp8", (256, 2, 1, 7956)),
    (5001, 4096, 700, "bf16", (256, 2, 1, 4096)),
    (5001, 4096, 500, "f32", (128, 2, 1, 5001)),
]


@pytest.mark.parametrize("size", LINEAR_SIZES, ids=lambda s: "x".join(map(str, s[:4])))
def test_forward_sizes_choose_their_kernels(gpu, size):
    M, N, K, kind, want = size
    got = linear_plan(gpu, M, N, K, kind, residual=True)
    assert all(w is None or g == w for g, w in zip(got, want)), got
    print(f"linear {M}x{N}x{K} {kind}", flush=True)
    linear_once(gpu, gpu.Stream(), np.random.default_rng(7), M, N, K, kind, "bf16", "gelu")


GRAD_SIZES = [  # M, N, K, type -> together, dw's tile and splits, dx's
    (8192, 4096, 2048, "bf16", (0, 128, 1, 256, 1)),
    (2000, 4000, 3000, "bf16", (1, 256, 1, 256, 1)),
    (2048, 8192, 2048, "bf16", (0, 256, 1, 128, 1)),
    (2000, 4000, 3000, "f32", (0, 128, 1, 64, 1)),
    (4100, 264, 2200, "bf16", (1, 128, 3, 128, 1)),
    (3000, 5000, 64, "f32", (0, 64, None, 64, None)),
]


@pytest.mark.parametrize("size", GRAD_SIZES, ids=lambda s: "x".join(map(str, s[:4])))
def test_gradient_sizes_choose_their_kernels(gpu, size):
    M, N, K, kind, want = size
    got = grad_plan(gpu, M, N, K, kind)
    assert all(w is None or g == w for g, w in zip(got, want)), got
    print(f"gradient {M}x{N}x{K} {kind}", flush=True)
    grad_once(gpu, gpu.Stream(), np.random.default_rng(8), M, N, K, kind, kind, "gelu")


# ---------------------------------------------------------------- the norm's rows
# Vectors of 16 bytes a row: one for each choice of waves and vectors a lane, at its
# ends, and the first length that is read twice.
VECTORS = [1, 2, 3, 64, 65, 128, 129, 192, 193, 256, 257, 384, 385, 512, 513, 768, 769, 1024, 1025,
           1536, 1537, 2048, 2049]


@pytest.mark.parametrize("vectors", VECTORS)
@pytest.mark.parametrize("kinds", ["f32 bf16", "bf16 fp8"])
def test_norm_rows_of_every_shape(gpu, kinds, vectors):
    xk, yk = kinds.split()
    V = 4 if xk == "f32" else 8
    rng, st = np.random.default_rng(vectors), gpu.Stream()
    for C in (vectors * V + V, vectors * V - V + 1, vectors * V - 1):
        if C < V:
            continue
        for M, pad, off in ((3, 0, 0), (9, 5, 1)):
            print(f"norm {kinds} {M}x{C}", flush=True)
            x, r = values(rng, (M, C), xk), values(rng, (M, C), xk)
            w = (1 + 0.2 * rng.standard_normal(C)).astype(np.float32).astype(np.float64)
            check_norm(gpu, st, x, r, w, xk, yk, 1e-6, f"{kinds} {M}x{C}", pad=pad, off=off)


@pytest.mark.parametrize("vectors", VECTORS)
@pytest.mark.parametrize("kinds", ["f32 bf16", "bf16 f32"])
def test_norm_gradient_rows_of_every_shape(gpu, kinds, vectors):
    xk, yk = kinds.split()
    V = 4 if xk == "f32" else 8
    rng, st = np.random.default_rng(vectors), gpu.Stream()
    for C, M in ((vectors * V + V, 5), (vectors * V - 1, 5), (vectors * V - V + 1, 300)):
        if C < V:
            continue
        print(f"norm gradient {kinds} {M}x{C}", flush=True)
        s, dy, ds = values(rng, (M, C), xk, 1.5), values(rng, (M, C), yk), values(rng, (M, C), xk)
        w = (1 + 0.2 * rng.standard_normal(C)).astype(np.float32).astype(np.float64)
        rstd = (1 / np.sqrt(np.mean(s * s, axis=1) + 1e-6)).astype(np.float32)
        DX = Mat(gpu, st, None, xk, 3, 1, (M, C))
        dweight = vector(gpu, st, np.full(C, np.nan))
        gpu.run_rmsnorm_grad_gpu(Mat(gpu, st, dy, yk, 1, 1).view, Mat(gpu, st, s, xk, 2, 0).view,
                                 vector(gpu, st, w), vector(gpu, st, rstd), DX.view, dweight,
                                 dsum=Mat(gpu, st, ds, xk).view, stream=st)
        st.sync()
        rd = rstd.astype(np.float64)[:, None]
        want, want_w = rms_norm_grad(dy, s, w, rd, ds)
        h, g = np.abs(s * rd), np.abs(dy * w)
        dot = np.sum(g * h, axis=1, keepdims=True) / C
        tol = 8 * EPS * (rd * (g + h * dot) + np.abs(want)) + rd * h * dot * (C + 4) * EPS
        close(DX.values(), want, tol + rounding(want, xk), f"dx {kinds} {M}x{C}")
        close(dweight.numpy(st), want_w, (M + 6) * EPS * np.sum(np.abs(dy) * h, axis=0) + 1e-30,
              "dweight")
