"""The dense operators around the sparse product, as measurable cases.

  norm    RMS norm of x + residual: f32, bf16, or 8-bit (e4m3) output with a
          scale per row; `dir` "forward" or "grad"
  linear  y = act(x W^T + bias) + residual on f32, bf16, or 8-bit (e4m3)
          operands with a scale per row; `dir` "forward" or "grad"
  adamw   one AdamW step over all tensors of a model, states in f32 or in
          e4m3 with a scale per 256 values

With `own` false, run() is the plain form in elementary torch operations in
32 bits; with `own` true it calls the library, whose buffers are the state's
torch tensors by address on the null stream (torch's current stream).
"""
from __future__ import annotations

import ctypes
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn}
_SIZE = {"f32": 4, "bf16": 2, "fp8": 1}
_FP8_MAX, _TINY, _BLOCK = 448.0, 1e-30, 256


def _package():
    name = "vcsr_spmm_amd"
    if name not in sys.modules:
        spec = importlib.util.spec_from_file_location(
            name, os.path.join(_ROOT, "vcsr-spmm_amd", "__init__.py"))
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
        mod.load_library()
    return sys.modules[name]


# ------------------------------------------------------------------- cases
def listed():
    return [
        # One new row through a served layer: the latency of a small call.
        dict(name="norm-row1-fp8", op="norm", dir="forward", M=1, C=4096, x="bf16", y="fp8",
             residual=True),
        # The banded 62K matrix's product at the headline width, f32 all
        # through: the sparse product's own output type.
        dict(name="norm-62k-o128-f32", op="norm", dir="forward", M=62451, C=128, x="f32",
             y="f32", residual=True),
        # A large batch before an 8-bit product.
        dict(name="norm-32k-fp8", op="norm", dir="forward", M=32768, C=4096, x="bf16", y="fp8",
             residual=True),
        # Training, a row length that is no multiple of a vector.
        dict(name="norm-grad-16k-bf16", op="norm", dir="grad", M=16384, C=2050, x="bf16",
             y="bf16", residual=True),
        # One row times a weight: the read of the weight.
        dict(name="linear-row1-bf16", op="linear", dir="forward", M=1, K=4096, N=4096, x="bf16",
             y="bf16", act="silu", residual=True),
        # Node features of the banded matrix, hidden width = input width.
        dict(name="linear-62k-o128-f32", op="linear", dir="forward", M=62451, K=128, N=128,
             x="f32", y="f32", act="gelu", residual=True),
        # The largest product: a batch through a wide hidden layer.
        dict(name="linear-8k-bf16", op="linear", dir="forward", M=8192, K=4096, N=8192, x="bf16",
             y="bf16", act="gelu", residual=False),
        # 8-bit serving of a ragged batch.
        dict(name="linear-5k-fp8", op="linear", dir="forward", M=5001, K=4096, N=4096, x="fp8",
             y="bf16", act="none", residual=True),
        # Training: all gradients of a layer; then of one with odd widths
        # (class scores of a graph) in f32.
        dict(name="linear-grad-8k-bf16", op="linear", dir="grad", M=8192, K=2048, N=4096,
             x="bf16", y="bf16", act="gelu", residual=False),
        dict(name="linear-grad-30k-f32", op="linear", dir="grad", M=30011, K=130, N=257, x="f32",
             y="f32", act="relu", residual=False),
        # The optimizer: a two-layer network on f32 states, and a model's
        # worth of tensors with 8-bit states and bf16 gradients.
        dict(name="adamw-2-layers-f32", op="adamw", layers=2, width=512, hidden=512, grad="f32",
             state="f32", copy=False, step=1),
        dict(name="adamw-24-layers-fp8", op="adamw", layers=24, width=1024, hidden=4096,
             grad="bf16", state="fp8", copy=True, step=1000),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A width: half of them multiples of 64 (where the range has some)."""
    w = _log_int(rng, lo, hi)
    if rng.random() < 0.5:
        w = min(hi, -(-w // 64) * 64)
    return w + 64 if w == 3072 else w


def draw(rng):
    """One more case: any operator, direction, type and size of the range."""
    op = rng.choice(["norm", "norm", "linear", "linear", "linear", "adamw"])
    if op == "adamw":
        width, hidden = _width(rng, 32, 1024), _width(rng, 32, 4096)
        most = max(1, min(24, 24 * 1024 * 4096 // (width * hidden)))
        return dict(op=op, layers=rng.randint(1, most), width=width, hidden=hidden,
                    grad=rng.choice(["f32", "bf16"]), state=rng.choice(["f32", "fp8", "fp8"]),
                    copy=rng.random() < 0.5, step=_log_int(rng, 1, 100000))
    way = rng.choice(["forward", "forward", "grad"])
    rows = _log_int(rng, 1, 65536) if rng.random() < 0.85 else rng.randint(1, 16)
    residual = rng.random() < 0.6
    if op == "norm":
        x = rng.choice(["f32", "bf16"])
        y = rng.choice(["f32", "bf16", "fp8"]) if way == "forward" else rng.choice(["f32", "bf16"])
        C = _width(rng, 8, 8192)
        while rows * C > 32768 * 4096:
            rows = max(1, rows // 2)
        return dict(op=op, dir=way, M=rows, C=C, x=x, y=y, residual=residual)
    x = rng.choice(["f32", "bf16", "bf16", "fp8"]) if way == "forward" else \
        rng.choice(["f32", "bf16"])
    y = "f32" if x == "f32" else rng.choice(["f32", "bf16", "bf16"])
    K, N = _width(rng, 8, 8192), _width(rng, 8, 8192)
    while rows * K * N > 8192 * 4096 * (8192 if way == "forward" else 2048) or \
            rows * max(K, N) > 32768 * 4096:
        rows = max(1, rows // 2)
    return dict(op=op, dir=way, M=rows, K=K, N=N, x=x, y=y,
                act=rng.choice(["none", "relu", "gelu", "silu"]), residual=residual)


# ------------------------------------------------------------------ inputs
class _Buf:
    """A torch tensor as the library's device buffers are described: bf16 as
    16-bit and e4m3 as 8-bit patterns."""

    _NP = {torch.float32: np.dtype(np.float32), torch.bfloat16: np.dtype(np.uint16),
           torch.float8_e4m3fn: np.dtype(np.uint8)}

    def __init__(self, t):
        self.t = t
        self.ptr = ctypes.c_void_p(t.data_ptr())
        self.nbytes = t.numel() * t.element_size()
        self.shape = tuple(t.shape)
        self.dtype = self._NP[t.dtype]


def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _to_fp8(y):
    """e4m3 values of the rows of `y` and their scales."""
    scale = y.abs().amax(dim=-1).clamp_min(_TINY) / _FP8_MAX
    return (y / scale[:, None]).to(torch.float8_e4m3fn), scale


def _tensors_of(case):
    """(name, shape, decays) of a model's parameters: per layer a norm's
    weight and two products with their biases."""
    w, h = case["width"], case["hidden"]
    one = [("norm", (w,), False), ("up", (h, w), True), ("up_bias", (h,), False),
           ("down", (w, h), True), ("down_bias", (w,), False)]
    return [(f"{i}.{n}", s, d) for i in range(case["layers"]) for n, s, d in one]


def _blocks(t):
    """The values of a tensor in rows of _BLOCK, the last one filled up."""
    flat = t.reshape(-1)
    return torch.nn.functional.pad(flat, (0, -flat.numel() % _BLOCK)).view(-1, _BLOCK)


def _state_to_fp8(t, never_zero):
    """e4m3 codes (the tensor's own shape) and scales of its blocks; with
    never_zero a nonzero value gets at least the smallest code."""
    b = _blocks(t)
    scale = b.abs().amax(dim=1).clamp_min(_TINY) / _FP8_MAX
    q = (b / scale[:, None]).to(torch.float8_e4m3fn)
    if never_zero:
        v = q.float()
        q = torch.where((v == 0) & (b > 0), torch.full_like(v, 2.0 ** -9), v).to(q.dtype)
    return q.view(-1)[:t.numel()].view(t.shape), scale


def _state_from_fp8(q, scale):
    b = _blocks(q.to(scale.dtype)) * scale[:, None]
    return b.view(-1)[:q.numel()].view(q.shape)


def _norm_inputs(case, seed):
    gen, M, C, xt = _generator(seed), case["M"], case["C"], _TORCH[case["x"]]
    # A residual stream: a few features carry much larger values.
    wide = torch.ones(C, device="cuda")
    wide[:: max(1, C // 8)] = 8.0
    x = (torch.randn((M, C), generator=gen, device="cuda") * wide).to(xt)
    s = dict(x=x, weight=1 + 0.1 * torch.randn(C, generator=gen, device="cuda"))
    if case["residual"]:
        s["residual"] = torch.randn((M, C), generator=gen, device="cuda").to(xt)
    if case["dir"] == "grad":
        s["dy"] = torch.randn((M, C), generator=gen, device="cuda").to(_TORCH[case["y"]])
        s["rstd"] = torch.rsqrt(x.float().square().mean(dim=1) + 1e-6)
    return s


def _linear_inputs(case, seed):
    gen, M, K, N, xt = _generator(seed), case["M"], case["K"], case["N"], _TORCH[case["x"]]

    def rand(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    s = {}
    if case["x"] == "fp8":
        s["x"], s["x_scale"] = _to_fp8(rand(M, K))
        s["w"], s["w_scale"] = _to_fp8(rand(N, K) / math.sqrt(K))
    else:
        s["x"], s["w"] = rand(M, K).to(xt), (rand(N, K) / math.sqrt(K)).to(xt)
    if case["dir"] == "grad":
        s["z"] = rand(M, N).to(_TORCH[case["y"]])
        s["dy"] = rand(M, N).to(_TORCH[case["y"]])
    else:
        s["bias"] = 0.1 * rand(N)
        if case["residual"]:
            s["residual"] = rand(M, N).to(_TORCH[case["y"]])
    return s


def _adamw_inputs(case, seed):
    gen, out = _generator(seed), []
    for name, shape, decays in _tensors_of(case):
        def rand():
            return torch.randn(shape, generator=gen, device="cuda")

        g = 1e-3 * rand()
        m = g * 0.3 + 3e-4 * rand() if case["step"] > 1 else torch.zeros_like(g)
        v = (1e-3 * rand()).square() * 0.5 + 5e-7 if case["step"] > 1 else torch.zeros_like(g)
        t = dict(name=name, decay=0.01 if decays else 0.0, grad=g.to(_TORCH[case["grad"]]),
                 param=0.02 * rand() if decays else 1 + 0.1 * rand())
        if case["state"] == "fp8":
            t["m"], t["m_scale"] = _state_to_fp8(m, False)
            t["v"], t["v_scale"] = _state_to_fp8(v.sqrt(), True)
        else:
            t["m"], t["v"] = m, v
        out.append(t)
    return out


_HYPER = dict(lr=1e-4, beta1=0.9, beta2=0.95, eps=1e-8, grad_scale=0.5)


def prepare(case, seed):
    s = dict(case=case)
    if case["op"] == "adamw":
        s["in"] = _adamw_inputs(case, seed)
        for t in s["in"]:
            if case["copy"]:
                t["copy"] = t["param"].to(torch.bfloat16)
        s["buf"] = [{k: _Buf(v) for k, v in t.items() if isinstance(v, torch.Tensor)}
                    for t in s["in"]]
        return s
    inputs = (_norm_inputs if case["op"] == "norm" else _linear_inputs)(case, seed)

    def new(shape, kind):
        return torch.empty(shape, dtype=_TORCH[kind], device="cuda")

    M, out = case["M"], {}
    if case["op"] == "norm" and case["dir"] == "forward":
        out["y"] = new((M, case["C"]), case["y"])
        out["rstd"] = new((M,), "f32")
        if case["y"] == "fp8":
            out["y_scale"] = new((M,), "f32")
        if case["residual"]:
            out["sum"] = new((M, case["C"]), case["x"])
    elif case["op"] == "norm":
        out["dx"], out["dweight"] = new((M, case["C"]), case["x"]), new((case["C"],), "f32")
    elif case["dir"] == "forward":
        out["y"] = new((M, case["N"]), case["y"])
    else:
        out["dx"], out["dw"] = new((M, case["K"]), case["x"]), new((case["N"], case["K"]), case["x"])
        out["dbias"] = new((case["N"],), "f32")
    s["in"], s["out"] = inputs, out
    s["buf"] = {k: _Buf(v) for k, v in {**inputs, **out}.items()}
    return s


# -------------------------------------------------------------- plain forms
def _act(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return z / (1 + torch.exp(-z)) if act == "silu" else z


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        t = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 0.134145 * z * z)
    if act == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    return torch.ones_like(z)


def _plain_norm(case, i):
    if case["dir"] == "grad":
        # x is the saved sum here; the residual's case has its gradient too.
        x, dy, r = i["x"].float(), i["dy"].float(), i["rstd"][:, None]
        xh, g = x * r, dy * i["weight"]
        dx = r * (g - xh * (g * xh).mean(dim=1, keepdim=True))
        if case["residual"]:
            dx = dx + i["residual"].float()
        return dict(dx=dx.to(i["x"].dtype), dweight=(dy * xh).sum(dim=0))
    t = i["x"].float()
    if case["residual"]:
        t = t + i["residual"].float()
    rstd = torch.rsqrt(t.square().mean(dim=1) + 1e-6)
    y = t * rstd[:, None] * i["weight"]
    out = dict(rstd=rstd)
    if case["residual"]:
        out["sum"] = t.to(i["x"].dtype)
    if case["y"] == "fp8":
        out["y"], out["y_scale"] = _to_fp8(y)
    else:
        out["y"] = y.to(_TORCH[case["y"]])
    return out


def _plain_linear(case, i):
    x, w = i["x"].float(), i["w"].float()
    if case["x"] == "fp8":
        x, w = x * i["x_scale"][:, None], w * i["w_scale"][:, None]
    if case["dir"] == "grad":
        dz = i["dy"].float() * _act_grad(i["z"].float(), case["act"])
        return dict(dx=torch.matmul(dz, w).to(i["x"].dtype),
                    dw=torch.matmul(dz.t(), x).to(i["x"].dtype), dbias=dz.sum(dim=0))
    y = _act(torch.matmul(x, w.t()) + i["bias"], case["act"])
    if case["residual"]:
        y = y + i["residual"].float()
    return dict(y=y.to(_TORCH[case["y"]]))


def _plain_adamw(case, tensors):
    h, t = _HYPER, case["step"]
    lr = h["lr"] / (1 - h["beta1"] ** t)
    root = 1 / math.sqrt(1 - h["beta2"] ** t)
    for e in tensors:
        g = e["grad"].float() * h["grad_scale"]
        if case["state"] == "fp8":
            m, v = _state_from_fp8(e["m"], e["m_scale"]), _state_from_fp8(e["v"], e["v_scale"])
            v = v * v
        else:
            m, v = e["m"], e["v"]
        m = m * h["beta1"] + g * (1 - h["beta1"])
        v = v * h["beta2"] + (g * g) * (1 - h["beta2"])
        r = v.sqrt()
        e["param"].copy_(e["param"] * (1 - h["lr"] * e["decay"]) - lr * (m / (r * root + h["eps"])))
        if case["state"] == "fp8":
            for k, value, never_zero in (("m", m, False), ("v", r, True)):
                q, scale = _state_to_fp8(value, never_zero)
                e[k].copy_(q)
                e[k + "_scale"].copy_(scale)
        else:
            e["m"].copy_(m)
            e["v"].copy_(v)
        if case["copy"]:
            e["copy"].copy_(e["param"])


# ------------------------------------------------------------------- passes
def _adamw_out(case, tensors):
    """What the step wrote, for the first layer and the last (a model has
    more tensors than are worth comparing)."""
    n = len(tensors) // case["layers"]
    keep = tensors if case["layers"] <= 2 else tensors[:n] + tensors[-n:]
    return {t["name"]: {k: v for k, v in t.items()
                        if k not in ("name", "decay", "grad")} for t in keep}


def _own_adamw(vs, s):
    if "plan" not in s:  # bound to the parameters once, as an optimizer is
        s["plan"] = vs.AdamW([dict(b, weight_decay=t["decay"]) for b, t in zip(s["buf"], s["in"])])
    s["plan"].step(step=s["case"]["step"], **_HYPER)


def _own(s):
    vs, case, b = _package(), s["case"], s["buf"]
    if case["op"] == "adamw":
        _own_adamw(vs, s)
        return None
    get = b.get
    if case["op"] == "norm" and case["dir"] == "forward":
        vs.run_rmsnorm_gpu(b["x"], b["weight"], b["y"], residual=get("residual"), sum=get("sum"),
                           y_scale=get("y_scale"), rstd=b["rstd"], eps=1e-6)
    elif case["op"] == "norm":
        vs.run_rmsnorm_grad_gpu(b["dy"], b["x"], b["weight"], b["rstd"], b["dx"], b["dweight"],
                                dsum=get("residual"))
    elif case["dir"] == "forward":
        vs.run_linear_gpu(b["x"], b["w"], b["y"], bias=b["bias"], residual=get("residual"),
                          act=case["act"], x_scale=get("x_scale"), w_scale=get("w_scale"))
    else:
        vs.run_linear_grad_gpu(b["dy"], b["x"], b["w"], z=b["z"], act=case["act"], dx=b["dx"],
                               dw=b["dw"], dbias=b["dbias"])
    return s["out"]


def run(state):
    case = state["case"]
    if own:
        out = _own(state)
    elif case["op"] == "adamw":
        out = _plain_adamw(case, state["in"])
    else:
        out = (_plain_norm if case["op"] == "norm" else _plain_linear)(case, state["in"])
    return _adamw_out(case, state["in"]) if case["op"] == "adamw" else out


def work(case):
    if case["op"] == "adamw":
        n = sum(math.prod(s) for _, s, _ in _tensors_of(case))
        scales = sum(-(-math.prod(s) // _BLOCK) for _, s, _ in _tensors_of(case))
        each = 8 + _SIZE[case["grad"]] + 4 * _SIZE[case["state"]] + (2 if case["copy"] else 0)
        return {"bytes": float(n * each + (16 * scales if case["state"] == "fp8" else 0)),
                "flops": 15.0 * n}
    M, xs, ys = case["M"], _SIZE[case["x"]], _SIZE[case["y"]]
    if case["op"] == "norm":
        C, r = case["C"], case["residual"]
        if case["dir"] == "forward":
            each = xs * (3 if r else 1) + ys
            rows = 4 + (4 if case["y"] == "fp8" else 0)
        else:
            each, rows = xs * (3 if r else 2) + ys, 4
        return {"bytes": float(M * C * each + M * rows + C * 8), "flops": 8.0 * M * C}
    K, N = case["K"], case["N"]
    if case["dir"] == "forward":
        return {"bytes": float((M + N) * K * xs + M * N * ys * (2 if case["residual"] else 1) + 4 * N
                               + (4 * (M + N) if case["x"] == "fp8" else 0)),
                "flops": 2.0 * M * N * K}
    return {"bytes": float(2 * (M + N) * K * xs + 2 * M * N * ys + 4 * N), "flops": 4.0 * M * N * K}


# ------------------------------------------------------------------ 64 bits
def _exact_norm(case, i):
    x, w = i["x"].double(), i["weight"].double()
    C = x.shape[1]
    if case["dir"] == "grad":
        dy, r = i["dy"].double(), i["rstd"].double().unsqueeze(1)
        # The Jacobian of s -> s * rstd(s), applied row by row.
        dot = torch.sum(dy * w * x, 1, keepdim=True)
        dx = r * dy * w - r.pow(3) * x * dot / C
        if case["residual"]:
            dx = dx + i["residual"].double()
        return dict(dx=dx, dweight=torch.sum(dy * x * r, 0))
    if case["residual"]:
        x = x + i["residual"].double()
    norm = torch.sqrt(torch.sum(x * x, 1) / C + 1e-6)
    y = w * x / norm.unsqueeze(1)
    out = dict(rstd=1 / norm)
    if case["residual"]:
        out["sum"] = x
    if case["y"] == "fp8":
        out["y_scale"] = torch.clamp(y.abs().max(1).values, min=_TINY) / _FP8_MAX
        y = y / out["y_scale"].unsqueeze(1)
    out["y"] = y
    return out


def _exact_linear(case, i):
    x, w = i["x"].to(torch.float32).double(), i["w"].to(torch.float32).double()
    if case["x"] == "fp8":
        x = x * i["x_scale"].double().view(-1, 1)
        w = w * i["w_scale"].double().view(-1, 1)

    def act(z):
        if case["act"] == "relu":
            return torch.where(z > 0, z, torch.zeros_like(z))
        if case["act"] == "gelu":
            # 0.5 (1 + tanh u) is the logistic function of 2u.
            return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
        return z * torch.sigmoid(z) if case["act"] == "silu" else z

    if case["dir"] == "forward":
        y = act(x @ w.T + i["bias"].double())
        return dict(y=y + i["residual"].double() if case["residual"] else y)
    z = i["z"].double().requires_grad_(True)
    with torch.enable_grad():
        dz, = torch.autograd.grad(act(z), z, i["dy"].double())
    return dict(dx=dz @ w, dw=dz.T.contiguous() @ x, dbias=dz.sum(0))


def _exact_adamw(case, tensors):
    h, n, out = _HYPER, case["step"], []
    for e in tensors:
        wide = {k: v.to(torch.float32).double() if isinstance(v, torch.Tensor) else v
                for k, v in e.items()}
        m, v = wide["m"], wide["v"]
        if case["state"] == "fp8":
            block = torch.arange(m.numel(), device=m.device).div(_BLOCK, rounding_mode="floor")
            m = m * wide["m_scale"][block].view(m.shape)
            v = (v * wide["v_scale"][block].view(m.shape)) ** 2
        g = wide["grad"] * h["grad_scale"]
        m = h["beta1"] * m + (1 - h["beta1"]) * g
        v = h["beta2"] * v + (1 - h["beta2"]) * g ** 2
        mhat, vhat = m / (1 - h["beta1"] ** n), v / (1 - h["beta2"] ** n)
        p = wide["param"] - h["lr"] * (mhat / (vhat.sqrt() + h["eps"]) + e["decay"] * wide["param"])
        t = dict(name=e["name"], decay=e["decay"], grad=None, param=p, m=m, v=v)
        if case["state"] == "fp8":
            for k, u in (("m", m), ("v", v.sqrt())):
                top = torch.zeros(int(block[-1]) + 1, dtype=torch.float64, device=u.device)
                top.scatter_reduce_(0, block, u.abs().view(-1), "amax")
                t[k + "_scale"] = torch.clamp(top, min=_TINY) / _FP8_MAX
                t[k] = u / t[k + "_scale"][block].view(u.shape)
        if case["copy"]:
            t["copy"] = p
        out.append(t)
    return out


def exact(case, seed):
    if case["op"] == "adamw":
        n = 5
        tensors = _adamw_inputs(case, seed)
        if case["layers"] > 2:
            tensors = tensors[:n] + tensors[-n:]
            case = dict(case, layers=2)
        return _adamw_out(case, _exact_adamw(case, tensors))
    if case["op"] == "norm":
        return _exact_norm(case, _norm_inputs(case, seed))
    return _exact_linear(case, _linear_inputs(case, seed))
