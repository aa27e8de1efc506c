"""A small residual graph network, trained and then served with this library.

Each of its layers aggregates over a sparse matrix A and mixes features with a
dense weight:

    t = A h + h                       run_vcsr_spmm_gpu_ex, run_rmsnorm_gpu (sum)
    u = t / rms(t) * g                run_rmsnorm_gpu, in bf16
    h = gelu(u W^T + b) + t           run_linear_gpu, W's bf16 copy

between an input layer and an output layer in FP32.  Training runs the
gradients of all of them (the sparse product's own is A^T's) and one AdamW step
over every tensor, 8-bit states for the weights; the loss is the mean square of
y - target, which the output layer writes directly (its residual is -target).
Serving runs the layers with 8-bit activations and weights.

    python3 examples/graph_layers.py [--nodes 4096] [--steps 60]
"""
from __future__ import annotations

import argparse
import importlib.util
import os
import sys

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def load_library_module():
    name = "vcsr_spmm_amd"
    if name not in sys.modules:
        spec = importlib.util.spec_from_file_location(
            name, os.path.join(ROOT, "vcsr-spmm_amd", "__init__.py"))
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    return sys.modules[name]


class Graph:
    """A (rows normalised) and A^T as uploaded formats."""

    def __init__(self, vs, rng, nodes, degree, st):
        rows = np.repeat(np.arange(nodes, dtype=np.int32), degree)
        cols = rng.integers(0, nodes, rows.size).astype(np.int32)
        vals = np.full(rows.size, 1.0 / degree, np.float32)
        self.fmt = vs.csr_to_vcsr_seg(
            vs.coo_to_csr(vs.Coo.from_arrays(nodes, nodes, rows, cols, vals)), 4, 64)
        self.fmt_t = vs.csr_to_vcsr_seg(
            vs.coo_to_csr(vs.Coo.from_arrays(nodes, nodes, cols, rows, vals)), 4, 64)
        self.fmt.upload(st)
        self.fmt_t.upload(st)


class Param:
    """A parameter with its gradient and optimizer states on the device."""

    def __init__(self, vs, st, value, grad, decay, bits8):
        n, up = value.size, lambda a: vs.DeviceArray.from_numpy(a, st)
        self.param, self.shape = up(value.astype(np.float32)), value.shape
        self.grad = vs.DeviceArray(value.shape, grad)
        self.decay, self.copy = decay, None
        if grad == vs.BF16:  # multiplied in bf16
            self.copy = up(vs.to_bf16(value))
        kind = vs.FP8 if bits8 else vs.F32
        self.m, self.v = (up(np.zeros(n, kind)) for _ in range(2))
        self.m_scale, self.v_scale = (
            (up(np.zeros(-(-n // 256), np.float32)) for _ in range(2)) if bits8 else (None, None))

    def entry(self):
        return dict(param=self.param, grad=self.grad, m=self.m, v=self.v, m_scale=self.m_scale,
                    v_scale=self.v_scale, copy=self.copy, weight_decay=self.decay)


class Network:
    def __init__(self, vs, st, rng, graph, nodes, n_in, width, n_out, layers):
        self.vs, self.st, self.graph, self.nodes, self.width = vs, st, graph, nodes, width

        def weight(n, k, grad):
            return Param(vs, st, rng.standard_normal((n, k)) / np.sqrt(k), grad, 0.01, True)

        def vector(n, value):
            return Param(vs, st, np.full(n, value), vs.F32, 0.0, False)

        self.w_in, self.b_in = weight(width, n_in, vs.F32), vector(width, 0.0)
        self.layers = [dict(g=vector(width, 1.0), w=weight(width, width, vs.BF16),
                            b=vector(width, 0.0)) for _ in range(layers)]
        self.w_out, self.b_out = weight(n_out, width, vs.F32), vector(n_out, 0.0)
        self.params = [self.w_in, self.b_in, self.w_out, self.b_out] + \
            [p for layer in self.layers for p in layer.values()]
        self.opt = vs.AdamW([p.entry() for p in self.params], st)

        def f32(cols=width):
            return vs.DeviceArray((nodes, cols), np.float32)

        def bf16():
            return vs.DeviceArray((nodes, width), vs.BF16)

        self.h = [f32() for _ in range(layers + 1)]
        self.z_in, self.err = f32(), f32(n_out)
        self.act = [dict(agg=f32(), t=f32(), u=bf16(), z=f32(),
                         rstd=vs.DeviceArray((nodes,), np.float32)) for _ in range(layers)]
        self.dh, self.dt, self.back, self.du = f32(), f32(), f32(), bf16()

    def forward(self, x, minus_target):
        """Leaves y - target in self.err."""
        vs, st, O = self.vs, self.st, self.width
        vs.run_linear_gpu(x, self.w_in.param, self.h[0], bias=self.b_in.param, act="relu",
                          z=self.z_in, stream=st)
        for i, (layer, a) in enumerate(zip(self.layers, self.act)):
            vs.run_vcsr_spmm_gpu_ex(self.graph.fmt, self.h[i], O, 0, a["agg"], st,
                                    accumulate=False)
            vs.run_rmsnorm_gpu(a["agg"], layer["g"].param, a["u"], residual=self.h[i], sum=a["t"],
                               rstd=a["rstd"], stream=st)
            vs.run_linear_gpu(a["u"], layer["w"].copy, self.h[i + 1], bias=layer["b"].param,
                              act="gelu", residual=a["t"], z=a["z"], stream=st)
        vs.run_linear_gpu(self.h[-1], self.w_out.param, self.err, bias=self.b_out.param,
                          residual=minus_target, stream=st)

    def backward(self, x):
        """Gradients of sum(err^2) / 2."""
        vs, st, O = self.vs, self.st, self.width
        vs.run_linear_grad_gpu(self.err, self.h[-1], self.w_out.param, dx=self.dh,
                               dw=self.w_out.grad, dbias=self.b_out.grad, stream=st)
        for layer, a in zip(reversed(self.layers), reversed(self.act)):
            vs.run_linear_grad_gpu(self.dh, a["u"], layer["w"].copy, z=a["z"], act="gelu",
                                   dx=self.du, dw=layer["w"].grad, dbias=layer["b"].grad,
                                   stream=st)
            vs.run_rmsnorm_grad_gpu(self.du, a["t"], layer["g"].param, a["rstd"], self.dt,
                                    layer["g"].grad, dsum=self.dh, stream=st)
            # t = A h + h: the gradient of h is dt + A^T dt.
            self.back.copy_from(self.dt, st)
            vs.run_vcsr_spmm_gpu(self.graph.fmt_t, self.dt, O, 0, self.back, st)
            self.dh, self.back = self.back, self.dh
        vs.run_linear_grad_gpu(self.dh, x, self.w_in.param, z=self.z_in, act="relu",
                               dw=self.w_in.grad, dbias=self.b_in.grad, stream=st)

    def serve(self, x):
        """The network with 8-bit activations and weights in its layers."""
        vs, st, n, O = self.vs, self.st, self.nodes, self.width
        h, agg, t = (vs.DeviceArray((n, O), np.float32) for _ in range(3))
        u, u_scale = vs.DeviceArray((n, O), vs.FP8), vs.DeviceArray((n,), np.float32)
        y = vs.DeviceArray(self.err.shape, np.float32)
        vs.run_linear_gpu(x, self.w_in.param, h, bias=self.b_in.param, act="relu", stream=st)
        for layer in self.layers:
            codes, scales = vs.quantize_fp8(layer["w"].param.numpy(st))
            w8, w_scale = (vs.DeviceArray.from_numpy(a, st) for a in (codes, scales))
            vs.run_vcsr_spmm_gpu_ex(self.graph.fmt, h, O, 0, agg, st, accumulate=False)
            vs.run_rmsnorm_gpu(agg, layer["g"].param, u, residual=h, sum=t, y_scale=u_scale,
                               stream=st)
            vs.run_linear_gpu(u, w8, h, bias=layer["b"].param, act="gelu", residual=t,
                              x_scale=u_scale, w_scale=w_scale, stream=st)
        vs.run_linear_gpu(h, self.w_out.param, y, bias=self.b_out.param, stream=st)
        st.sync()
        return y.numpy(st)


def train(nodes=4096, degree=16, n_in=48, width=128, n_out=10, layers=2, steps=60, say=print):
    """Trains on targets made by a fixed graph function; returns the losses, the
    trained network's outputs and those of its 8-bit form."""
    vs = load_library_module()
    vs.load_library()
    rng, st = np.random.default_rng(0), vs.Stream()
    graph = Graph(vs, rng, nodes, degree, st)
    feats = rng.standard_normal((nodes, n_in)).astype(np.float32)
    target = np.tanh(feats @ (rng.standard_normal((n_in, n_out)) / np.sqrt(n_in)))
    x = vs.DeviceArray.from_numpy(feats, st)
    minus_target = vs.DeviceArray.from_numpy((-target).astype(np.float32), st)
    net = Network(vs, st, rng, graph, nodes, n_in, width, n_out, layers)
    losses = []
    for step in range(1, steps + 1):
        net.forward(x, minus_target)
        net.backward(x)
        net.opt.step(step, lr=2e-3, beta2=0.95, grad_scale=2.0 / target.size, stream=st)
        if step == 1 or step % 10 == 0:
            st.sync()
            losses.append(float(np.mean(net.err.numpy(st) ** 2)))
            say(f"step {step:4d}  loss {losses[-1]:.5f}")
    net.forward(x, minus_target)
    st.sync()
    y = net.err.numpy(st) + target
    y8 = net.serve(x)
    say(f"8-bit serving: {np.linalg.norm(y8 - y) / np.linalg.norm(y):.3%} from the bf16 network")
    return losses, y, y8


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--nodes", type=int, default=4096)
    ap.add_argument("--steps", type=int, default=60)
    args = ap.parse_args()
    train(nodes=args.nodes, steps=args.steps, say=lambda s: print(s, flush=True))
