"""The embedding's gradient of more tokens than are ranked, sorted by digits, on the GPU:
types, widths, strides and tables of one to four digits.  Each size is held to that sort."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from block_ref import rounding, values
from conftest import capture, hip_runtime
from dense_ref import EPS, Mat, close
from embed_plans import DIGITS, RANKS, embed_grad_plan
from test_gpu_embed import GRAD, grad_once, ints, tokens

pytestmark = pytest.mark.gpu


def by_digits(vs, M, V, C, dk, tk, add, digits=None):
    plan = embed_grad_plan(vs, M, V, C, dk, tk, add)
    assert plan[0] == DIGITS and digits in (None, plan[1]), plan


@pytest.mark.parametrize("C", [1, 4, 9, 64, 129, 257, 520, 1030])
@pytest.mark.parametrize("kinds", GRAD)
def test_embed_grad_by_digits(gpu, kinds, C):
    """On both sides of the sort's limit; digits of 3 to 9 bits."""
    dk, tk = kinds.split()
    st, rng = gpu.Stream(), np.random.default_rng(C)
    assert embed_grad_plan(gpu, 12288, 60, C, dk, tk)[0] == RANKS
    for n, (M, V, kind) in enumerate([(12288, 60, "runs"), (12289, 60, "runs"),
                                      (12289, 7, "uniform"), (13001, 7000, "frequent"),
                                      (16385, 3, "same"), (20000, 513, "frequent"),
                                      (20011, 400, "runs"), (12300, 40, "outside")]):
        pad, off = ((0, 0), (8, 0), (3, 1))[n % 3]
        print(f"embed grad digits {kinds} C={C} M={M} V={V} {kind}", flush=True)
        for add in (n % 2 == 0, n % 2 == 1) if C in (9, 520) else (n % 2 == 0,):
            if n:
                by_digits(gpu, M, V, C, dk, tk, add)
            grad_once(gpu, st, rng, M, V, C, dk, tk, tokens(rng, M, V, kind), add, pad, off)


@pytest.mark.parametrize("V, digits", [(1, 1), (2, 1), (255, 1), (256, 1), (511, 1), (512, 2),
                                       (513, 2), (1023, 2), (1024, 2), (262143, 2), (262144, 3),
                                       (300000, 3)])
@pytest.mark.parametrize("kind", ["uniform", "frequent", "sorted", "backwards"])
def test_embed_grad_by_digits_of_a_table(gpu, V, digits, kind):
    st, rng = gpu.Stream(), np.random.default_rng(V)
    for M in (12289, 13300):
        by_digits(gpu, M, V, 8, "bf16", "f32", False, digits)
        ids = tokens(rng, M, V, kind if kind == "frequent" else "uniform")
        ids[:3], ids[-3:] = V - 1, 0
        ids = {"sorted": np.sort(ids), "backwards": np.sort(ids)[::-1]}.get(kind, ids)
        print(f"embed grad digits M={M} V={V} {kind}", flush=True)
        one = grad_once(gpu, st, np.random.default_rng(1), M, V, 8, "bf16", "f32", ids, False)
        two = grad_once(gpu, st, np.random.default_rng(1), M, V, 8, "bf16", "f32", ids, False)
        assert one.tobytes() == two.tobytes()


@pytest.mark.parametrize("V, digits", [((1 << 27) - 1, 3), (1 << 27, 4), ((1 << 31) - 1, 4)])
def test_embed_grad_by_four_digits(gpu, V, digits):
    """The rows of a table of up to 2^31 - 1 rows that have tokens, which are all that an
    accumulating call touches."""
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(6)
    table = vs.DeviceArray((V, 1), vs.BF16)
    lib = vs.load_library()
    for M in (12289, 40000):
        by_digits(vs, M, V, 1, "bf16", "bf16", True, digits)
        vs._check(lib.vcsr_memset_d(table.ptr, 0, table.nbytes, st.h))
        some = np.concatenate([[0, 1, V - 1, V - 2, V // 2, V // 2 + 1, (1 << 24) + 1, (1 << 16) - 1,
                                255, 256, 511, 512], rng.integers(0, V, 200)])
        ids = rng.choice(some, M)
        ids[:4], ids[-3:] = (-1, V, V - 1, 0), (V - 1, -(1 << 31), 0)
        dy = values(rng, (M, 1), "bf16")
        print(f"embed grad of a table of {V} rows M={M}", flush=True)
        vs.run_embed_grad_gpu(Mat(vs, st, dy, "bf16").view, ints(vs, st, ids), table,
                              accumulate=True, stream=st)
        st.sync()
        got = np.empty(1, np.uint16)
        for v in np.unique(some):
            vs._check(lib.vcsr_memcpy_d2h(got.ctypes.data, table.ptr.value + int(v) * 2, 2, st.h))
            mine = ids == v
            want = dy[mine].sum()
            # A run of n tokens rounds n sums, the product with its scale and the sum of it
            # and the row once each.
            tol = (mine.sum() + 2) * EPS * np.abs(dy[mine]).sum() + rounding(want, "bf16")
            close((got.astype(np.uint32) << 16).view(np.float32)[0], want, tol, f"row {v}")


def test_embed_grad_by_digits_replayed_from_a_graph(gpu):
    """Three digits, written over the table and added to it, on other tokens each replay."""
    vs, st = gpu, gpu.Stream()
    hip = hip_runtime()
    rng = np.random.default_rng(12)
    M, V, C = 12289, 263000, 16
    by_digits(vs, M, V, C, "bf16", "f32", False, 3)
    DY = Mat(vs, st, values(rng, (M, C), "bf16"), "bf16")
    D = vs.DeviceArray((V, C), np.float32)
    ids = ints(vs, st, tokens(rng, M, V, "frequent"))

    def step():
        vs.run_embed_grad_gpu(DY.view, ids, D, stream=st)
        vs.run_embed_grad_gpu(DY.view, ids, D, scale=0.5, accumulate=True, stream=st)

    step()
    graph, kinds = capture(hip, st, step)
    gexec = ctypes.c_void_p()
    try:
        assert kinds and all(k == 0 for k in kinds), kinds  # kernels only
        assert hip.hipGraphInstantiateWithFlags(ctypes.byref(gexec), graph, 0) == 0
        for n in range(3):
            ids.copy_from(ints(vs, st, tokens(rng, M, V, ("frequent", "same", "uniform")[n])), st)
            step()
            st.sync()
            eager = D.numpy(st).tobytes()
            vs._check(vs.load_library().vcsr_memset_d(D.ptr, 0x5B, D.nbytes, st.h))
            st.sync()
            print(f"replay {n}", flush=True)
            assert hip.hipGraphLaunch(gexec, st.h) == 0
            st.sync()
            same = D.numpy(st).tobytes() == eager
            assert same, n
    finally:
        if gexec.value:
            hip.hipGraphExecDestroy(gexec)
        hip.hipGraphDestroy(graph)
