"""One training step of a small network through the operators together, as a program runs
them, against its formulas in 64 bits: tokens to rows (embedding), layer norm, gated
projection, linear layer back onto the residual stream, output by the table itself
(whose gradient the embedding's is added to), all gradients, and the optimizer."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from block_ref import layer_norm, values
from conftest import capture, hip_runtime
from dense_ref import act, act_grad

pytestmark = pytest.mark.gpu


class Net:
    """V tokens, width C, hidden width H; FP32 all through or bf16 operands."""

    def __init__(self, vs, st, rng, M, V, C, H, kind):
        self.vs, self.st, self.M, self.kind = vs, st, M, kind
        self.scale = float(np.float32(np.sqrt(C)))
        T = vs.BF16 if kind == "bf16" else vs.F32
        self.host = dict(table=values(rng, (V, C), kind, C ** -0.5), gain=1 + 0.1 * values(rng, C, "f32"),
                         shift=0.1 * values(rng, C, "f32"), wg=values(rng, (H, C), kind, C ** -0.5),
                         wu=values(rng, (H, C), kind, C ** -0.5), wd=values(rng, (C, H), kind, H ** -0.5))
        self.host = {k: v.astype(np.float32).astype(np.float64) for k, v in self.host.items()}

        def up(a, t):
            a = np.ascontiguousarray(a, np.float32)
            return vs.DeviceArray.from_numpy(vs.to_bf16(a) if t == vs.BF16 else a, st)

        # bf16 networks keep FP32 parameters and a copy to multiply with, as AdamW writes it.
        self.par = {k: up(v, vs.F32) for k, v in self.host.items()}
        self.use = {k: up(v, T) if v.ndim == 2 else self.par[k] for k, v in self.host.items()}
        self.grad = {k: vs.DeviceArray(v.shape, T if v.ndim == 2 else vs.F32)
                     for k, v in self.host.items()}
        zeros = {k: [up(np.zeros(v.shape), vs.F32) for _ in range(2)] for k, v in self.host.items()}
        self.opt = vs.AdamW([dict(param=self.par[k], grad=self.grad[k], m=zeros[k][0], v=zeros[k][1],
                                  copy=self.use[k] if kind == "bf16" and v.ndim == 2 else None)
                             for k, v in self.host.items()], st)

        def new(rows, cols, t=T):
            return vs.DeviceArray((rows, cols), t)

        self.x, self.u, self.s = new(M, C), new(M, C), new(M, C)
        self.zg, self.zu, self.h, self.dh = (new(M, H) for _ in range(4))
        self.du, self.ds, self.dx = new(M, C), new(M, C), new(M, C)
        self.logits, self.dlogits = new(M, V), None
        self.mean, self.rstd = (vs.DeviceArray((M,), np.float32) for _ in range(2))

    def step(self, ids, dlogits, n=None):
        vs, st, w, g = self.vs, self.st, self.use, self.grad
        vs.run_embed_gpu(w["table"], ids, self.x, scale=self.scale, stream=st)
        vs.run_layernorm_gpu(self.x, w["gain"], self.u, bias=w["shift"], mean=self.mean,
                             rstd=self.rstd, stream=st)
        vs.run_gated_gpu(self.u, w["wg"], w["wu"], self.h, z_gate=self.zg, z_up=self.zu, stream=st)
        vs.run_linear_gpu(self.h, w["wd"], self.s, residual=self.x, stream=st)
        vs.run_linear_gpu(self.s, w["table"], self.logits, stream=st)
        # Back: the table's gradient from the output layer, then the embedding's on top.
        vs.run_linear_grad_gpu(dlogits, self.s, w["table"], dx=self.ds, dw=g["table"], stream=st)
        vs.run_linear_grad_gpu(self.ds, self.h, w["wd"], dx=self.dh, dw=g["wd"], stream=st)
        vs.run_gated_grad_gpu(self.dh, self.u, w["wg"], w["wu"], self.zg, self.zu, dx=self.du,
                              dw_gate=g["wg"], dw_up=g["wu"], stream=st)
        vs.run_layernorm_grad_gpu(self.du, self.x, w["gain"], self.mean, self.rstd, self.dx,
                                  g["gain"], g["shift"], dsum=self.ds, stream=st)
        vs.run_embed_grad_gpu(self.dx, ids, g["table"], scale=self.scale, accumulate=True, stream=st)
        if n is not None:
            self.opt.step(n, lr=1e-2, stream=st)

    def gradients(self):
        self.st.sync()
        out = {}
        for k, b in self.grad.items():
            a = b.numpy(self.st)
            out[k] = (self.vs.from_bf16(a) if a.dtype == np.uint16 else a).astype(np.float64)
        return out


def formulas(p, ids, dlogits, scale):
    """All gradients of <dlogits, logits> in 64 bits."""
    V = p["table"].shape[0]
    inside = (ids >= 0) & (ids < V)
    x = np.where(inside[:, None], p["table"][np.where(inside, ids, 0)], 0) * scale
    _, mean, rstd, u = layer_norm(x, None, p["gain"], p["shift"], float(np.float32(1e-5)))
    zg, zu = u @ p["wg"].T, u @ p["wu"].T
    h = act(zg, "silu") * zu
    s = h @ p["wd"].T + x
    ds, table = dlogits @ p["table"], dlogits.T @ s
    dh, wd = ds @ p["wd"], ds.T @ h
    dg, du_ = dh * zu * act_grad(zg, "silu"), dh * act(zg, "silu")
    du, wg, wu = dg @ p["wg"] + du_ @ p["wu"], dg.T @ u, du_.T @ u
    hat, g = (x - mean) * rstd, du * p["gain"]
    dx = ds + rstd * (g - g.mean(1, keepdims=True) - hat * (g * hat).mean(1, keepdims=True))
    np.add.at(table, ids[inside], scale * dx[inside])
    return dict(table=table, gain=(du * hat).sum(0), shift=du.sum(0), wg=wg, wu=wu, wd=wd)


def ints(vs, st, a):
    return vs.DeviceArray.from_numpy(np.ascontiguousarray(a, np.int32), st)


@pytest.mark.parametrize("M, V, C, H", [(1, 40, 64, 96), (200, 90, 128, 257), (1100, 700, 72, 192),
                                        (700, 50, 130, 130)])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_a_block_trains(gpu, kind, M, V, C, H):
    vs, st = gpu, gpu.Stream()
    rng = np.random.default_rng(M + V)
    net = Net(vs, st, rng, M, V, C, H, kind)
    ids = rng.integers(-1, V, M).astype(np.int32)
    dlogits = values(rng, (M, V), kind, 1 / M)
    print(f"block {kind} M={M} V={V} C={C} H={H}", flush=True)
    dev = vs.DeviceArray.from_numpy(
        vs.to_bf16(dlogits) if kind == "bf16" else dlogits.astype(np.float32), st)
    net.step(ints(vs, st, ids), dev)
    want = formulas(net.host, ids, dlogits, net.scale)
    # Of each gradient's norm.  Its path has at most 12 results that are rounded to the
    # type one after the other, u = 2^-8 or 2^-24 each, and sums of at most n = 1100 terms;
    # what enters a product comes out grown by its condition, at most 4 here (sums of random
    # signs: the norms of factors and result differ by no more).
    tol = {"bf16": 12 * 2.0 ** -8, "f32": 12 * 2.0 ** -24 * 40}[kind]
    for k, got in net.gradients().items():
        off = np.linalg.norm(got - want[k]) / np.linalg.norm(want[k])
        print(f"  {k}: {off:.2e}", flush=True)
        assert off <= tol, (k, off, tol)
    # The step itself: parameters move against their gradient, and bf16 copies follow.
    net.opt.step(1, lr=1e-2, stream=st)
    st.sync()
    for k, v in net.host.items():
        new = net.par[k].numpy(st).astype(np.float64)
        grad = net.gradients()[k]
        some = np.abs(grad) > 1e-6
        assert np.all((new - v)[some] * grad[some] < 0), k
        if kind == "bf16" and v.ndim == 2:
            assert np.array_equal(net.use[k].numpy(st), vs.to_bf16(new.astype(np.float32))), k


def test_a_block_from_a_graph(gpu):
    """The whole step captured: replays on other tokens give the bits of eager calls."""
    vs, st = gpu, gpu.Stream()
    hip = hip_runtime()
    rng = np.random.default_rng(3)
    M, V, C, H = 300, 120, 96, 200
    net = Net(vs, st, rng, M, V, C, H, "bf16")
    ids = ints(vs, st, rng.integers(-1, V, M))
    dev = vs.DeviceArray.from_numpy(vs.to_bf16(values(rng, (M, V), "bf16", 1 / M)), st)
    net.step(ids, dev)
    st.sync()
    graph, kinds = capture(hip, st, lambda: net.step(ids, dev))
    gexec = ctypes.c_void_p()
    try:
        assert kinds and all(k == 0 for k in kinds), kinds
        assert hip.hipGraphInstantiateWithFlags(ctypes.byref(gexec), graph, 0) == 0
        for n in range(3):
            ids.copy_from(ints(vs, st, rng.integers(-1, V, M)), st)
            net.step(ids, dev)
            eager = {k: v.tobytes() for k, v in net.gradients().items()}
            for b in net.grad.values():
                b.zero(st)
            st.sync()
            print(f"replay {n}", flush=True)
            assert hip.hipGraphLaunch(gexec, st.h) == 0
            same = {k: v.tobytes() for k, v in net.gradients().items()} == eager
            assert same, n
    finally:
        if gexec.value:
            hip.hipGraphExecDestroy(gexec)
        hip.hipGraphDestroy(graph)


def test_blocks_on_two_streams(gpu):
    """Two networks on streams of their own at the same time: the bits of one after the
    other."""
    vs = gpu
    nets, want = [], []
    for k in range(2):
        st, rng = vs.Stream(), np.random.default_rng(50 + k)
        M, V, C, H = 2000, 300, 128, 256
        net = Net(vs, st, rng, M, V, C, H, "bf16")
        ids = ints(vs, st, rng.integers(-1, V, M))
        dev = vs.DeviceArray.from_numpy(vs.to_bf16(values(rng, (M, V), "bf16", 1 / M)), st)
        net.step(ids, dev)
        want.append({k: v.tobytes() for k, v in net.gradients().items()})
        nets.append((net, ids, dev))
    for _ in range(3):
        for net, ids, dev in nets:
            net.step(ids, dev)
    for (net, _, _), w in zip(nets, want):
        same = {k: v.tobytes() for k, v in net.gradients().items()} == w
        assert same
