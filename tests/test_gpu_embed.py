"""The embedding and its gradient on the GPU against their formulas in 64 bits.

Tolerances: a product of FP32 values rounds once (u), one with an 8-bit row's scale
twice; a run of n tokens is added in chains of at most n terms, each rounding its sum."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import scipy.sparse

from block_ref import rounding, values
from conftest import capture, hip_runtime
from dense_ref import EPS, NP, Mat, close, vector

pytestmark = pytest.mark.gpu


def ints(vs, st, a):
    return vs.DeviceArray.from_numpy(np.ascontiguousarray(a, np.int32), st)


def tokens(rng, M, V, kind):
    """Ids of a distribution, some of them outside the table."""
    if kind == "same":
        return np.full(M, V // 2, np.int32)
    if kind == "outside":
        return rng.choice(np.int32([-1, V, -(1 << 31), (1 << 31) - 1]), M).astype(np.int32)
    if kind == "frequent":  # the k-th most frequent about 1 / k as often as the first
        ids = np.exp(rng.random(M) * np.log(V + 1)).astype(np.int64) - 1
        ids = rng.permutation(V)[np.clip(ids, 0, V - 1)]
    elif kind == "runs":  # of all lengths around a chunk's
        ids = np.repeat(rng.permutation(V), rng.choice([1, 2, 7, 8, 9, 15, 16, 17, 31, 33, 63, 64,
                                                        65, 127, 128, 129, 200], V))[:M]
        ids = np.concatenate([ids, rng.integers(0, V, M - len(ids))])
        ids = rng.permutation(ids)
    else:
        ids = rng.integers(0, V, M)
    return np.where(rng.random(M) < 0.05, rng.choice([-1, V, V + 7], M), ids).astype(np.int32)


FORWARD = ["f32 f32", "f32 bf16", "bf16 f32", "bf16 bf16", "fp8 f32", "fp8 bf16"]


@pytest.mark.parametrize("C", [1, 3, 8, 15, 16, 17, 64, 129, 257, 520, 1030, 2050, 8200])
@pytest.mark.parametrize("kinds", FORWARD)
def test_embed(gpu, kinds, C):
    xk, yk = kinds.split()
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(C)
    for M, V, pad, off in ((1, 1, 0, 0), (5, 3, 3, 1), (70, 300, 16, 0), (1001, 40, 1, 2)):
        print(f"embed {kinds} C={C} M={M} V={V} pad={pad} off={off}", flush=True)
        table, ids = values(rng, (V, C), xk), tokens(rng, M, V, "uniform")
        ts = (0.5 + rng.random(V)).astype(np.float32) if xk == "fp8" else None
        T, Y = Mat(vs, st, table, xk, pad, off), Mat(vs, st, None, yk, pad, 2 * off, (M, C))
        vs.run_embed_gpu(T.view, ints(vs, st, ids), Y.view, scale=1.7,
                         table_scale=vector(vs, st, ts) if ts is not None else None, stream=st)
        st.sync()
        want = np.float64(np.float32(1.7)) * table
        if ts is not None:
            want = want * ts.astype(np.float64)[:, None]
        inside = (ids >= 0) & (ids < V)
        want = np.where(inside[:, None], want[np.where(inside, ids, 0)], 0)
        close(Y.values(), want, 2.01 * EPS * np.abs(want) + rounding(want, yk), f"{kinds} {M}x{C}")
        assert not Y.values()[~inside].any()


@pytest.mark.parametrize("C", [2, 4, 5, 6, 7, 9, 12, 13, 20, 31])
@pytest.mark.parametrize("kinds", FORWARD)
def test_embed_of_narrow_rows(gpu, kinds, C):
    """Around the vectors of 4, 8 and 16 values that the pairs of types have."""
    xk, yk = kinds.split()
    vs, st, rng = gpu, gpu.Stream(), np.random.default_rng(C)
    for M, V, pad, off in ((3, 2, 0, 0), (300, 50, 1, 1), (65, 7, 4, 3)):
        table, ids = values(rng, (V, C), xk), tokens(rng, M, V, "uniform")
        ts = np.full(V, 0.5, np.float32) if xk == "fp8" else None
        T, Y = Mat(vs, st, table, xk, pad, off), Mat(vs, st, None, yk, pad, 2 * off, (M, C))
        vs.run_embed_gpu(T.view, ints(vs, st, ids), Y.view, scale=2.0,
                         table_scale=vector(vs, st, ts) if ts is not None else None, stream=st)
        st.sync()
        want = table * (1 if ts is not None else 2)  # exact in FP32
        inside = (ids >= 0) & (ids < V)
        want = np.where(inside[:, None], want[np.where(inside, ids, 0)], 0)
        close(Y.values(), want, rounding(want, yk), f"{kinds} {M}x{C}")


@pytest.mark.parametrize("kinds", FORWARD)
def test_embed_of_a_large_result(gpu, kinds):
    """128 MB of y and more, which go past the caches; whole rows and others."""
    xk, yk = kinds.split()
    vs, st, rng = gpu, gpu.Stream(), np.random.default_rng(6)
    V, M = 3000, 1 << 17
    for C in (512, 516, 509) if yk == "bf16" else (256, 260, 253):
        table = values(rng, (V, C), "fp8" if xk == "fp8" else "bf16")  # exact in y's type
        ids = tokens(rng, M, V, "uniform")
        ts = np.ones(V, np.float32) if xk == "fp8" else None
        y = vs.DeviceArray((M, C), vs.BF16 if yk == "bf16" else np.float32)
        print(f"embed {kinds} of {M} x {C}", flush=True)
        vs.run_embed_gpu(Mat(vs, st, table, xk).view, ints(vs, st, ids), y,
                         table_scale=vector(vs, st, ts) if ts is not None else None, stream=st)
        st.sync()
        inside = (ids >= 0) & (ids < V)
        rows = np.vstack([table, np.zeros((1, C))]).astype(np.float32)
        want = (vs.to_bf16(rows) if yk == "bf16" else rows)[np.where(inside, ids, V)]
        assert np.array_equal(y.numpy(st), want)


def test_embed_keeps_what_is_not_finite(gpu):
    """NaN and infinities in the table's rows; a row of zeros for padding whatever row 0
    holds."""
    vs, st = gpu, gpu.Stream()
    for kind in ("f32", "bf16"):
        table = np.ones((4, 70))
        table[0], table[1, 3], table[2, 69] = np.nan, np.inf, -np.inf
        ids = np.int32([-1, 0, 1, 2, 3, 4, 1])
        Y = Mat(vs, st, None, kind, shape=(7, 70))
        vs.run_embed_gpu(Mat(vs, st, table, kind).view, ints(vs, st, ids), Y.view, scale=2.0,
                         stream=st)
        st.sync()
        want = np.where(((ids >= 0) & (ids < 4))[:, None], 2 * table[ids % 4], 0)
        close(Y.values(), want, 0, kind)


def test_embed_of_many_tokens(gpu):
    """More rows than a block has; a table past 4 GiB read at both ends."""
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(2)
    V, C = 70001, 16400
    big = vs.DeviceArray((V, C), np.float32)
    big.zero(st)
    lib, rows = vs.load_library(), [0, 1, 32768, 65470, 65471, V - 1]
    x = rng.standard_normal((len(rows), C)).astype(np.float32)
    for r, v in zip(rows, x):
        vs._check(lib.vcsr_memcpy_h2d(big.ptr.value + r * C * 4, v.ctypes.data, v.nbytes, st.h))
    ids = np.int32([rows[i] for i in (5, 0, 3, 3, 4, 1, 2)] + [40000])
    Y = Mat(vs, st, None, "f32", shape=(8, C))
    print("a large table", flush=True)
    vs.run_embed_gpu(big, ints(vs, st, ids), Y.view, stream=st)
    st.sync()
    y = Y.values()
    assert np.array_equal(y[:7], x[[5, 0, 3, 3, 4, 1, 2]].astype(np.float64)) and not y[7].any()
    del big
    M, V, C = (1 << 22) + 5, 1000, 4
    table, ids = values(rng, (V, C), "bf16"), tokens(rng, M, V, "uniform")
    out = vs.DeviceArray((M, C), np.float32)
    vs.run_embed_gpu(Mat(vs, st, table, "bf16").view, ints(vs, st, ids), out, stream=st)
    st.sync()
    inside = (ids >= 0) & (ids < V)
    same = np.array_equal(out.numpy(st), np.where(inside[:, None], table[np.where(inside, ids, 0)], 0))
    assert same


GRAD = ["f32 f32", "bf16 f32", "f32 bf16", "bf16 bf16"]  # dy, dtable


def grad_once(vs, st, rng, M, V, C, dk, tk, ids, accumulate, pad=0, off=0, scale=0.75):
    dy = values(rng, (M, C), dk)
    base = values(rng, (V, C), tk) if accumulate else None
    DY = Mat(vs, st, dy, dk, pad, off)
    T = Mat(vs, st, base, tk, pad, 2 * off, (V, C))
    vs.run_embed_grad_gpu(DY.view, ints(vs, st, ids), T.view, scale=scale, accumulate=accumulate,
                          stream=st)
    st.sync()
    kept = np.flatnonzero((ids >= 0) & (ids < V))
    hot = scipy.sparse.csr_matrix((np.ones(len(kept)), (ids[kept], kept)), shape=(V, M))
    n = np.bincount(ids[kept], minlength=V)[:, None]
    want = scale * (hot @ dy) + (base if accumulate else 0)
    tol = (n + 1) * EPS * scale * (hot @ np.abs(dy)) + EPS * np.abs(want)
    what = f"{dk} {tk} M={M} V={V} C={C}"
    got = T.values()
    close(got, want, np.where(n > 0, tol + rounding(want, tk), 0), what)
    return T.codes()


@pytest.mark.parametrize("C", [1, 4, 9, 64, 129, 257, 520, 1030])
@pytest.mark.parametrize("kinds", GRAD)
def test_embed_grad(gpu, kinds, C):
    """Numbers of tokens around what is sorted in a wave, by ranks and by digits."""
    dk, tk = kinds.split()
    st, rng = gpu.Stream(), np.random.default_rng(C)
    for n, (M, V, kind) in enumerate([(1, 1, "uniform"), (2, 9, "same"), (63, 5, "uniform"),
                                      (64, 100, "frequent"), (65, 7, "frequent"),
                                      (130, 2, "uniform"), (1000, 50, "runs"),
                                      (3000, 40, "runs"), (5001, 7000, "frequent"),
                                      (8192, 3, "frequent"), (8193, 60, "runs"),
                                      (12000, 513, "frequent")]):
        print(f"embed grad {kinds} C={C} M={M} V={V} {kind}", flush=True)
        pad, off = ((0, 0), (8, 0), (3, 1))[n % 3]
        ids = tokens(rng, M, V, kind)
        grad_once(gpu, st, rng, M, V, C, dk, tk, ids, n % 2 == 0, pad, off)


@pytest.mark.parametrize("kind", ["same", "outside", "uniform", "frequent", "sorted", "backwards"])
@pytest.mark.parametrize("M", [1, 40, 64, 65, 700, 8192, 8200, 40000])
def test_embed_grad_distributions(gpu, kind, M):
    st, rng = gpu.Stream(), np.random.default_rng(M)
    V, C = 600, 72
    ids = tokens(rng, M, V, "frequent" if kind in ("sorted", "backwards") else kind)
    ids = {"sorted": np.sort(ids), "backwards": np.sort(ids)[::-1]}.get(kind, ids)
    for dk, tk, add in (("bf16", "f32", False), ("f32", "bf16", True)):
        print(f"embed grad {kind} M={M} {dk} {tk}", flush=True)
        one = grad_once(gpu, st, np.random.default_rng(1), M, V, C, dk, tk, ids, add)
        two = grad_once(gpu, st, np.random.default_rng(1), M, V, C, dk, tk, ids, add)
        assert one.tobytes() == two.tobytes()


@pytest.mark.parametrize("M", [12288, 12289, 12800, 12801, 16384, 16385, 65536, 65537, 131072,
                               131073, 262145, 524288, 524289])
def test_embed_grad_tiles(gpu, M):
    """Numbers of tokens at both ends of the sort's tiles and of their number."""
    st, rng = gpu.Stream(), np.random.default_rng(M)
    for V, kind in ((40, "runs"), (70000, "frequent")):
        print(f"embed grad tiles M={M} V={V}", flush=True)
        grad_once(gpu, st, rng, M, V, 4, "f32", "f32", tokens(rng, M, V, kind), False)


@pytest.mark.parametrize("C", [1, 3, 7, 8, 9, 40, 63, 64, 65, 255, 256, 500, 511, 513, 4100])
@pytest.mark.parametrize("tk", ["f32", "bf16"])
def test_embed_grad_clears_rows(gpu, tk, C):
    """Rows shorter and longer than a wave's pieces, most of them without a token, in
    whole groups and a last one of fewer."""
    st, rng = gpu.Stream(), np.random.default_rng(C)
    for n, (M, V) in enumerate([(20, 1000), (90, 1024), (13000, 641), (3, 63), (66, 65)]):
        pad, off = ((0, 0), (8, 0), (3, 1))[n % 3]
        print(f"embed grad clears {tk} C={C} M={M} V={V} pad={pad}", flush=True)
        ids = rng.choice(np.array([0, 1, V // 2, V - 1, V, -1]), M).astype(np.int32)
        grad_once(gpu, st, rng, M, V, C, "bf16", tk, ids, False, pad, off)


@pytest.mark.parametrize("V", [1, 2, 255, 256, 511, 512, 513, 1023, 1024, 262143, 262144, 300000])
def test_embed_grad_digits(gpu, V):
    """Tables of one, two and three digits' rows, at both ends of each."""
    st, rng = gpu.Stream(), np.random.default_rng(V)
    for M in (8300, 30000):
        ids = tokens(rng, M, V, "uniform")
        ids[:3], ids[-3:] = V - 1, 0
        print(f"embed grad digits M={M} V={V}", flush=True)
        grad_once(gpu, st, rng, M, V, 8, "bf16", "f32", ids, False)


def test_embed_grad_ids_of_31_bits(gpu):
    """Four digits: the rows of a table of 2^31 - 1 rows that have tokens, which are all
    that an accumulating call touches."""
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(6)
    V = (1 << 31) - 1
    table = vs.DeviceArray((V, 1), vs.BF16)
    lib = vs.load_library()
    for M in (50, 3000, 9000):
        vs._check(lib.vcsr_memset_d(table.ptr, 0, table.nbytes, st.h))
        some = np.concatenate([[0, 1, V - 1, V - 2, 1 << 30, (1 << 24) + 1],
                               rng.integers(0, V, 40)])
        ids = rng.choice(some, M)
        ids[:4] = -1, V, V - 1, 0
        dy = values(rng, (M, 1), "bf16")
        print(f"embed grad of a table of 2^31 rows M={M}", flush=True)
        vs.run_embed_grad_gpu(Mat(vs, st, dy, "bf16").view, ints(vs, st, ids), table,
                              accumulate=True, stream=st)
        st.sync()
        got = np.empty(1, np.uint16)
        for v in some:
            vs._check(lib.vcsr_memcpy_d2h(got.ctypes.data, table.ptr.value + int(v) * 2, 2, st.h))
            mine = ids == v
            mine &= ids < V
            want = dy[mine].sum()
            tol = (mine.sum() + 2) * EPS * np.abs(dy[mine]).sum() + rounding(want, "bf16")
            close((got.astype(np.uint32) << 16).view(np.float32)[0], want, tol, f"row {v}")


@pytest.mark.parametrize("M, V, C", [(300000, 1000, 16), (131073, 131072, 8), (70000, 33, 40)])
def test_embed_grad_of_many_tokens(gpu, M, V, C):
    st, rng = gpu.Stream(), np.random.default_rng(M)
    print(f"embed grad M={M} V={V} C={C}", flush=True)
    grad_once(gpu, st, rng, M, V, C, "bf16", "f32", tokens(rng, M, V, "frequent"), False)
    grad_once(gpu, st, rng, M, V, C, "f32", "f32", np.full(M, V - 1, np.int32), True)


def test_embed_grad_keeps_nan_in_its_rows(gpu):
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(8)
    for M in (60, 4000):
        V, C = 30, 100
        ids = tokens(rng, M, V, "uniform")
        ids[0], ids[1], ids[2] = 3, 5, -1
        dy = values(rng, (M, C), "f32")
        dy[0, 7], dy[1, 99], dy[2, 0] = np.nan, np.inf, np.nan
        T = Mat(vs, st, None, "f32", shape=(V, C))
        vs.run_embed_grad_gpu(Mat(vs, st, dy, "f32").view, ints(vs, st, ids), T.view, stream=st)
        st.sync()
        got = T.values()
        assert np.isnan(got[3, 7]) and got[5, 99] == np.inf
        assert np.isfinite(np.delete(got.ravel(), [3 * C + 7, 5 * C + 99])).all()


def test_embed_grad_of_no_tokens(gpu):
    """Zeros, or with accumulate nothing."""
    vs, st = gpu, gpu.Stream()
    one = np.ones((5, 9))
    none, dy = vs.DeviceView(0, (0,), np.int32), vs.DeviceView(0, (0, 9), vs.F32)
    for add in (False, True):
        T = Mat(vs, st, one, "bf16", 3, 1)
        vs.run_embed_grad_gpu(dy, none, T.view, accumulate=add, stream=st)
        st.sync()
        assert np.array_equal(T.values(), one if add else 0 * one)
    vs.run_embed_gpu(T.view, none, dy, stream=st)


def test_embed_grad_against_differences(gpu):
    """The lookup is linear in the table: <dy, y(table + t v)> changes by t <dtable, v>."""
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(10)
    M, V, C = 40, 11, 24
    ids, dy, v = tokens(rng, M, V, "uniform"), values(rng, (M, C), "f32"), values(rng, (V, C), "f32")
    Y, T = Mat(vs, st, None, "f32", shape=(M, C)), Mat(vs, st, None, "f32", shape=(V, C))
    vs.run_embed_gpu(Mat(vs, st, v, "f32").view, ints(vs, st, ids), Y.view, scale=3.5, stream=st)
    vs.run_embed_grad_gpu(Mat(vs, st, dy, "f32").view, ints(vs, st, ids), T.view, scale=3.5,
                          stream=st)
    st.sync()
    terms = dy * Y.values()
    assert abs(terms.sum() - (T.values() * v).sum()) <= 2.0 ** -20 * np.abs(terms).sum()


@pytest.mark.parametrize("M", [50, 2000, 20000])
def test_embed_replayed_from_a_graph(gpu, M):
    """Lookup and gradient captured, replayed between eager calls on other tokens."""
    vs, st = gpu, gpu.Stream()
    hip = hip_runtime()
    rng = np.random.default_rng(12)
    V, C = 300, 136
    T, DY = Mat(vs, st, values(rng, (V, C), "bf16"), "bf16"), \
        Mat(vs, st, values(rng, (M, C), "bf16"), "bf16")
    Y, D = Mat(vs, st, None, "f32", shape=(M, C)), Mat(vs, st, None, "f32", shape=(V, C))
    ids = ints(vs, st, tokens(rng, M, V, "frequent"))

    def step():
        vs.run_embed_gpu(T.view, ids, Y.view, scale=2.0, stream=st)
        vs.run_embed_grad_gpu(DY.view, ids, D.view, scale=2.0, stream=st)

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
            eager = Y.codes().tobytes(), D.codes().tobytes()
            for m in (Y, D):
                m.buf.copy_from(vs.DeviceArray.from_numpy(m.host, st), st)
            st.sync()
            print(f"replay {n}", flush=True)
            assert hip.hipGraphLaunch(gexec, st.h) == 0
            st.sync()
            same = (Y.codes().tobytes(), D.codes().tobytes()) == eager
            assert same, n
    finally:
        if gexec.value:
            hip.hipGraphExecDestroy(gexec)
        hip.hipGraphDestroy(graph)


@pytest.mark.parametrize("kinds", ["f32 f32", "bf16 f32", "f32 bf16", "bf16 bf16", "fp8 f32",
                                   "fp8 bf16"])
def test_embed_of_large_results(gpu, kinds):
    """y of 128 MB and more, written past the caches: every value."""
    xk, yk = kinds.split()
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(21)
    M, V, C = (1 << 17) + 3, 500, 512
    table, ids = values(rng, (V, C), xk), tokens(rng, M, V, "uniform")
    ts = (0.5 + rng.random(V)).astype(np.float32) if xk == "fp8" else None
    out = vs.DeviceArray((M, C), NP[yk])
    print(f"embed large {kinds}", flush=True)
    vs.run_embed_gpu(Mat(vs, st, table, xk).view, ints(vs, st, ids), out,
                     table_scale=vector(vs, st, ts) if ts is not None else None, stream=st)
    st.sync()
    # Each row of the table once, and that all of y's rows are theirs bit for bit.
    rows = vs.DeviceArray((V + 1, C), NP[yk])
    vs.run_embed_gpu(Mat(vs, st, table, xk).view, ints(vs, st, np.arange(V + 1)), rows,
                     table_scale=vector(vs, st, ts) if ts is not None else None, stream=st)
    st.sync()
    inside = (ids >= 0) & (ids < V)
    same = np.array_equal(out.numpy(st), rows.numpy(st)[np.where(inside, ids, V)])
    assert same


def test_embed_grad_of_a_large_table(gpu):
    """Zeros of 128 MB and more, past the caches, beside the rows of few and of many
    tokens."""
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(22)
    V, C = 70000, 512
    for M in (20, 700, 20000):
        ids = tokens(rng, M, V, "frequent")
        dy = values(rng, (M, C), "bf16")
        out = vs.DeviceArray((V, C), np.float32)
        vs._check(vs.load_library().vcsr_memset_d(out.ptr, 0x5B, out.nbytes, st.h))
        print(f"embed grad large M={M}", flush=True)
        vs.run_embed_grad_gpu(Mat(vs, st, dy, "bf16").view, ints(vs, st, ids), out, stream=st)
        st.sync()
        got = out.numpy(st)
        met = np.unique(ids[(ids >= 0) & (ids < V)])
        one = vs.DeviceArray((V, C), np.float32)
        one.zero(st)
        vs.run_embed_grad_gpu(Mat(vs, st, dy, "bf16").view, ints(vs, st, ids), one,
                              accumulate=True, stream=st)
        st.sync()
        same = np.array_equal(got, one.numpy(st))
        assert same
        want = np.stack([dy[ids == v].sum(0) for v in met[:200]])
        size = np.stack([np.abs(dy[ids == v]).sum(0) for v in met[:200]])
        n = np.array([(ids == v).sum() for v in met[:200]])[:, None]
        close(got[met[:200]], want, (n + 2) * EPS * size, "rows with tokens")
        got[met] = 0
        assert not got.any()
