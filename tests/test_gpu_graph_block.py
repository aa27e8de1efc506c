"""The sparse product together with the embedding, layer norm, gated projection and linear
layer on one stream, as a layer of a graph network runs them, against its formulas in 64
bits: forward, all gradients (the sparse product's by its transpose), captured and replayed.

    x = scale * table[ids]          run_embed_gpu
    t = A x + x                     run_vcsr_spmm_gpu_ex, run_layernorm_gpu (sum)
    u = layer norm of t             run_layernorm_gpu
    h = silu(u Wg^T) * (u Wu^T)     run_gated_gpu
    y = h Wd^T + t                  run_linear_gpu
"""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import scipy.sparse

from block_ref import layer_norm, values
from conftest import capture, hip_runtime
from dense_ref import act, act_grad

pytestmark = pytest.mark.gpu

DEGREE = 12


class Layer:
    """M nodes, a table of V rows, width C, hidden width H.  FP32 between the sparse product
    and the norm; the products' operands in FP32 or bf16."""

    def __init__(self, vs, st, rng, M, V, C, H, kind):
        self.vs, self.st, self.M, self.C = vs, st, M, C
        self.scale = float(np.float32(np.sqrt(C)))
        T = vs.BF16 if kind == "bf16" else vs.F32
        rows = np.repeat(np.arange(M, dtype=np.int32), DEGREE)
        cols = rng.integers(0, M, rows.size).astype(np.int32)
        vals = (rng.random(rows.size) / DEGREE).astype(np.float32)
        self.A = scipy.sparse.coo_matrix((vals.astype(np.float64), (rows, cols)), (M, M)).tocsr()
        self.fmt, self.fmt_t = (
            vs.csr_to_vcsr_seg(vs.coo_to_csr(vs.Coo.from_arrays(M, M, r, c, vals)), 4, 64)
            for r, c in ((rows, cols), (cols, rows)))
        for f in (self.fmt, self.fmt_t):
            f.upload(st)
        host = dict(table=values(rng, (V, C), "f32", C ** -0.5),
                    gain=1 + 0.1 * values(rng, C, "f32"), shift=0.1 * values(rng, C, "f32"),
                    wg=values(rng, (H, C), kind, C ** -0.5), wu=values(rng, (H, C), kind, C ** -0.5),
                    wd=values(rng, (C, H), kind, H ** -0.5))
        self.host = {k: v.astype(np.float32).astype(np.float64) for k, v in host.items()}

        def up(k, v):
            v = np.ascontiguousarray(v, np.float32)
            return vs.DeviceArray.from_numpy(vs.to_bf16(v) if k[0] == "w" and T == vs.BF16 else v, st)

        self.par = {k: up(k, v) for k, v in self.host.items()}
        self.grad = {k: vs.DeviceArray(v.shape, T if k[0] == "w" else vs.F32)
                     for k, v in self.host.items()}

        def new(cols, t=vs.F32):
            return vs.DeviceArray((M, cols), t)

        self.x, self.agg, self.t, self.y = (new(C) for _ in range(4))
        self.u, self.du = new(C, T), new(C, T)
        self.zg, self.zu, self.h, self.dh = (new(H, T) for _ in range(4))
        self.dt, self.back = new(C), new(C)
        self.mean, self.rstd = (vs.DeviceArray((M,), np.float32) for _ in range(2))

    def step(self, ids, dy):
        vs, st, p, g, C = self.vs, self.st, self.par, self.grad, self.C
        vs.run_embed_gpu(p["table"], ids, self.x, scale=self.scale, stream=st)
        vs.run_vcsr_spmm_gpu_ex(self.fmt, self.x, C, 0, self.agg, st, accumulate=False)
        vs.run_layernorm_gpu(self.agg, p["gain"], self.u, bias=p["shift"], residual=self.x,
                             sum=self.t, mean=self.mean, rstd=self.rstd, stream=st)
        vs.run_gated_gpu(self.u, p["wg"], p["wu"], self.h, z_gate=self.zg, z_up=self.zu, stream=st)
        vs.run_linear_gpu(self.h, p["wd"], self.y, residual=self.t, stream=st)
        vs.run_linear_grad_gpu(dy, self.h, p["wd"], dx=self.dh, dw=g["wd"], stream=st)
        vs.run_gated_grad_gpu(self.dh, self.u, p["wg"], p["wu"], self.zg, self.zu, dx=self.du,
                              dw_gate=g["wg"], dw_up=g["wu"], stream=st)
        vs.run_layernorm_grad_gpu(self.du, self.t, p["gain"], self.mean, self.rstd, self.dt,
                                  g["gain"], g["shift"], dsum=dy, stream=st)
        # What reaches x: dt itself, and A^T dt on top of it in the table.
        vs.run_vcsr_spmm_gpu_ex(self.fmt_t, self.dt, C, 0, self.back, st, accumulate=False)
        vs.run_embed_grad_gpu(self.dt, ids, g["table"], scale=self.scale, stream=st)
        vs.run_embed_grad_gpu(self.back, ids, g["table"], scale=self.scale, accumulate=True,
                              stream=st)

    def results(self):
        self.st.sync()
        out = {"y": self.y.numpy(self.st), **{k: b.numpy(self.st) for k, b in self.grad.items()}}
        return {k: (self.vs.from_bf16(a) if a.dtype == np.uint16 else a).astype(np.float64)
                for k, a in out.items()}

    def formulas(self, ids, dy):
        p, A, V = self.host, self.A, self.host["table"].shape[0]
        inside = (ids >= 0) & (ids < V)
        x = np.where(inside[:, None], p["table"][np.where(inside, ids, 0)], 0) * self.scale
        t, mean, rstd, u = layer_norm(A @ x, x, p["gain"], p["shift"], float(np.float32(1e-5)))
        zg, zu = u @ p["wg"].T, u @ p["wu"].T
        h = act(zg, "silu") * zu
        dh = dy @ p["wd"]
        dg, dv = dh * zu * act_grad(zg, "silu"), dh * act(zg, "silu")
        du = dg @ p["wg"] + dv @ p["wu"]
        hat, g = (t - mean) * rstd, du * p["gain"]
        dt = dy + rstd * (g - g.mean(1, keepdims=True) - hat * (g * hat).mean(1, keepdims=True))
        dx, table = dt + A.T @ dt, np.zeros_like(p["table"])
        np.add.at(table, ids[inside], self.scale * dx[inside])
        return dict(y=h @ p["wd"].T + t, table=table, gain=(du * hat).sum(0), shift=du.sum(0),
                    wg=dg.T @ u, wu=dv.T @ u, wd=dy.T @ h)


def ints(vs, st, a):
    return vs.DeviceArray.from_numpy(np.ascontiguousarray(a, np.int32), st)


@pytest.mark.parametrize("M, V, C, H", [(300, 300, 32, 64), (1500, 200, 64, 257),
                                        (1100, 700, 130, 96), (13000, 4000, 16, 48)])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_a_graph_layer_trains(gpu, kind, M, V, C, H):
    vs, st, rng = gpu, gpu.Stream(), np.random.default_rng(M + V)
    layer = Layer(vs, st, rng, M, V, C, H, kind)
    ids = rng.integers(-1, V, M).astype(np.int32)
    dy = values(rng, (M, C), "f32", 1 / M)
    print(f"graph layer {kind} M={M} V={V} C={C} H={H}", flush=True)
    layer.step(ints(vs, st, ids), vs.DeviceArray.from_numpy(dy.astype(np.float32), st))
    want = layer.formulas(ids, dy)
    # Of each result's norm.  A path has at most 12 results that are rounded to the type one
    # after the other, u = 2^-8 or 2^-24 each, and sums whose errors grow with the root of
    # their n <= 13000 terms at most (random signs: 114 u); what enters a product comes out
    # grown by its condition, at most 4 here.
    tol = {"bf16": 12 * 2.0 ** -8, "f32": 4 * (12 + 114) * 2.0 ** -24}[kind]
    for k, got in layer.results().items():
        off = np.linalg.norm(got - want[k]) / np.linalg.norm(want[k])
        print(f"  {k}: {off:.2e}", flush=True)
        assert off <= tol, (k, off, tol)


@pytest.mark.parametrize("M, V, C, H", [(900, 400, 64, 96), (13000, 500, 24, 32)])
def test_a_graph_layer_from_a_graph(gpu, M, V, C, H):
    """The whole step captured: replays on other tokens, between eager calls, give their
    bits (the sparse product's kernel adds without atomics)."""
    vs, st, rng = gpu, gpu.Stream(), np.random.default_rng(3)
    hip = hip_runtime()
    layer = Layer(vs, st, rng, M, V, C, H, "bf16")
    ids = ints(vs, st, rng.integers(-1, V, M))
    dy = vs.DeviceArray.from_numpy(values(rng, (M, C), "f32", 1 / M).astype(np.float32), st)
    layer.step(ids, dy)
    st.sync()
    graph, kinds = capture(hip, st, lambda: layer.step(ids, dy))
    gexec = ctypes.c_void_p()
    try:
        assert kinds and all(k == 0 for k in kinds), kinds
        assert hip.hipGraphInstantiateWithFlags(ctypes.byref(gexec), graph, 0) == 0
        for n in range(3):
            ids.copy_from(ints(vs, st, rng.integers(-1, V, M)), st)
            layer.step(ids, dy)
            eager = {k: v.tobytes() for k, v in layer.results().items()}
            for b in (layer.y, *layer.grad.values()):
                b.zero(st)
            st.sync()
            print(f"replay {n}", flush=True)
            assert hip.hipGraphLaunch(gexec, st.h) == 0
            same = {k: v.tobytes() for k, v in layer.results().items()} == eager
            assert same, n
    finally:
        if gexec.value:
            hip.hipGraphExecDestroy(gexec)
        hip.hipGraphDestroy(graph)


def test_graph_layers_on_two_streams(gpu):
    """Two layers on streams of their own at the same time: the bits of one after the other."""
    vs, runs, want = gpu, [], []
    for k in range(2):
        st, rng = vs.Stream(), np.random.default_rng(50 + k)
        M, V, C, H = 3000 + 500 * k, 300, 64, 128
        layer = Layer(vs, st, rng, M, V, C, H, "bf16")
        ids = ints(vs, st, rng.integers(-1, V, M))
        dy = vs.DeviceArray.from_numpy(values(rng, (M, C), "f32", 1 / M).astype(np.float32), st)
        layer.step(ids, dy)
        want.append({n: v.tobytes() for n, v in layer.results().items()})
        runs.append((layer, ids, dy))
    for _ in range(3):
        for layer, ids, dy in runs:
            layer.step(ids, dy)
    for (layer, _, _), w in zip(runs, want):
        same = {n: v.tobytes() for n, v in layer.results().items()} == w
        assert same
