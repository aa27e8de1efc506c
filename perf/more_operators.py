"""Three operators of a network's block, as measurable cases.

  embed      y = scale * table[ids] on f32, bf16, or 8-bit (e4m3, a scale per
             row) tables; `dir` "forward" or "grad", the latter written over a
             gradient or added to one
  layernorm  layer norm of x + residual: f32, bf16, or 8-bit (e4m3) output with
             a scale per row; `dir` "forward" or "grad"
  gated      y = act(x Wg^T + bg) * (x Wu^T + bu) on f32, bf16, or 8-bit (e4m3)
             operands with a scale per row; `dir` "forward" or "grad"

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
_FP8_MAX, _TINY, _EPS = 448.0, 1e-30, 1e-5


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
        # One new token of a served network: the latency of a small call.
        dict(name="embed-row1-fp8", op="embed", dir="forward", M=1, V=32768, C=4096, x="fp8",
             y="bf16"),
        # A large batch's tokens.
        dict(name="embed-64k-bf16", op="embed", dir="forward", M=65536, V=65536, C=2048, x="bf16",
             y="bf16"),
        # Its gradient in training, the whole table's written anew.
        dict(name="embed-grad-32k-bf16", op="embed", dir="grad", M=32768, V=32768, C=2048,
             x="f32", y="bf16", accumulate=False),
        # Odd sizes, added to the gradient of an output layer that shares the table.
        dict(name="embed-grad-5k-f32-add", op="embed", dir="grad", M=5001, V=50001, C=257,
             x="f32", y="f32", accumulate=True),
        # One new row through a served layer, before an 8-bit product.
        dict(name="layernorm-row1-fp8", op="layernorm", dir="forward", M=1, C=4096, x="bf16",
             y="fp8", residual=True),
        # The banded 62K matrix's product at the headline width, f32 all
        # through: the sparse product's own output type.
        dict(name="layernorm-62k-o128-f32", op="layernorm", dir="forward", M=62451, C=128, x="f32",
             y="f32", residual=True),
        # Training, a row length that is no multiple of a vector.
        dict(name="layernorm-grad-16k-bf16", op="layernorm", dir="grad", M=16384, C=2050, x="bf16",
             y="bf16", residual=True),
        # One row times two weights: the read of the weights.
        dict(name="gated-row1-bf16", op="gated", dir="forward", M=1, K=4096, N=8192, x="bf16",
             y="bf16", act="silu", save=False, bias=False),
        # The largest product: a training batch, both products' results kept
        # for the gradient.
        dict(name="gated-8k-bf16", op="gated", dir="forward", M=8192, K=4096, N=8192, x="bf16",
             y="bf16", act="silu", save=True, bias=False),
        # 8-bit serving of a ragged batch.
        dict(name="gated-5k-fp8", op="gated", dir="forward", M=5001, K=4096, N=4096, x="fp8",
             y="bf16", act="gelu", save=False, bias=True),
        # Training: all gradients of a block; then of one with odd widths
        # (node features of a graph) in f32.
        dict(name="gated-grad-8k-bf16", op="gated", dir="grad", M=8192, K=2048, N=4096, x="bf16",
             y="bf16", act="silu", bias=False),
        dict(name="gated-grad-30k-f32", op="gated", dir="grad", M=30011, K=130, N=257, x="f32",
             y="f32", act="gelu", bias=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A width: half of them multiples of 64 (where the range has some)."""
    w = _log_int(rng, lo, hi)
    return min(hi, -(-w // 64) * 64) if rng.random() < 0.5 else w


def draw(rng):
    """One more case: any operator, direction, type and size of the range."""
    op = rng.choice(["embed", "embed", "layernorm", "layernorm", "gated", "gated", "gated"])
    way = rng.choice(["forward", "grad"])
    rows = _log_int(rng, 1, 65536) if rng.random() < 0.85 else rng.randint(1, 16)
    wide = rng.choice(["f32", "bf16"])
    if op == "embed":
        C, V = _width(rng, 8, 8192), _log_int(rng, 2, 131072)
        while rows * C > 65536 * 2048:
            rows = max(1, rows // 2)
        while V * C > 65536 * 2048:
            V = max(2, V // 2)
        if way == "forward":
            return dict(op=op, dir=way, M=rows, V=V, C=C, x=rng.choice(["f32", "bf16", "fp8"]),
                        y=wide)
        return dict(op=op, dir=way, M=rows, V=V, C=C, x=rng.choice(["f32", "bf16"]), y=wide,
                    accumulate=rng.random() < 0.5)
    if op == "layernorm":
        C = _width(rng, 8, 8192)
        while rows * C > 32768 * 4096:
            rows = max(1, rows // 2)
        y = rng.choice(["f32", "bf16", "fp8"]) if way == "forward" else rng.choice(["f32", "bf16"])
        return dict(op=op, dir=way, M=rows, C=C, x=wide, y=y, residual=rng.random() < 0.6)
    x = rng.choice(["f32", "bf16", "bf16", "fp8"]) if way == "forward" else wide
    y = "f32" if x == "f32" else rng.choice(["f32", "bf16", "bf16"])
    K, N = _width(rng, 8, 8192), _width(rng, 8, 8192)
    while rows * K * N > 8192 * 4096 * (8192 if way == "forward" else 2048) or \
            rows * max(K, N) > 16384 * 4096:
        rows = max(1, rows // 2)
    case = dict(op=op, dir=way, M=rows, K=K, N=N, x=x, y=y,
                act=rng.choice(["none", "relu", "gelu", "silu"]), bias=rng.random() < 0.5)
    return dict(case, save=rng.random() < 0.5) if way == "forward" else case


# ------------------------------------------------------------------ inputs
class _Buf:
    """A torch tensor as the library's device buffers are described: bf16 as
    16-bit and e4m3 as 8-bit patterns."""

    _NP = {torch.float32: np.dtype(np.float32), torch.bfloat16: np.dtype(np.uint16),
           torch.float8_e4m3fn: np.dtype(np.uint8), torch.int32: np.dtype(np.int32)}

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


def _scale(case):
    return math.sqrt(case["C"])


def _ids(gen, M, V):
    """Tokens as text has them: the k-th most frequent about 1 / k as often as
    the first, those ranks spread over the table; one in 32 is padding (-1)."""
    u = torch.rand(M, generator=gen, device="cuda", dtype=torch.float64)
    rank = (torch.exp(u * math.log(V + 1)) - 1).long().clamp_(0, V - 1)
    ids = torch.randperm(V, generator=gen, device="cuda")[rank]
    pad = torch.rand(M, generator=gen, device="cuda") < 1 / 32
    return torch.where(pad, torch.full_like(ids, -1), ids).to(torch.int32)


def _embed_inputs(case, seed):
    gen, M, V, C = _generator(seed), case["M"], case["V"], case["C"]
    s = dict(ids=_ids(gen, M, V))
    if case["dir"] == "grad":
        s["dy"] = torch.randn((M, C), generator=gen, device="cuda").to(_TORCH[case["y"]])
        if case["accumulate"]:
            s["dtable"] = torch.randn((V, C), generator=gen, device="cuda").to(_TORCH[case["x"]])
        return s
    table = torch.randn((V, C), generator=gen, device="cuda") / _scale(case)
    if case["x"] == "fp8":
        s["table"], s["table_scale"] = _to_fp8(table)
    else:
        s["table"] = table.to(_TORCH[case["x"]])
    return s


def _norm_inputs(case, seed):
    gen, M, C, xt = _generator(seed), case["M"], case["C"], _TORCH[case["x"]]
    # A residual stream: a few features carry much larger values, and rows have
    # a mean of their own.
    wide = torch.ones(C, device="cuda")
    wide[:: max(1, C // 8)] = 8.0
    x = torch.randn((M, C), generator=gen, device="cuda") * wide
    x = (x + torch.randn((M, 1), generator=gen, device="cuda")).to(xt)
    s = dict(x=x, weight=1 + 0.1 * torch.randn(C, generator=gen, device="cuda"))
    if case["residual"]:
        s["residual"] = torch.randn((M, C), generator=gen, device="cuda").to(xt)
    if case["dir"] == "grad":
        s["dy"] = torch.randn((M, C), generator=gen, device="cuda").to(_TORCH[case["y"]])
        s["mean"] = x.float().mean(dim=1)
        s["rstd"] = torch.rsqrt((x.float() - s["mean"][:, None]).square().mean(dim=1) + _EPS)
    else:
        s["bias"] = 0.1 * torch.randn(C, generator=gen, device="cuda")
    return s


def _gated_inputs(case, seed):
    gen, M, K, N, xt = _generator(seed), case["M"], case["K"], case["N"], _TORCH[case["x"]]

    def rand(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    s = {}
    if case["x"] == "fp8":
        s["x"], s["x_scale"] = _to_fp8(rand(M, K))
        s["w_gate"], s["gate_scale"] = _to_fp8(rand(N, K) / math.sqrt(K))
        s["w_up"], s["up_scale"] = _to_fp8(rand(N, K) / math.sqrt(K))
    else:
        s["x"] = rand(M, K).to(xt)
        s["w_gate"], s["w_up"] = ((rand(N, K) / math.sqrt(K)).to(xt) for _ in range(2))
    if case["dir"] == "grad":
        s["z_gate"], s["z_up"], s["dy"] = (rand(M, N).to(_TORCH[case["y"]]) for _ in range(3))
    elif case["bias"]:
        s["gate_bias"], s["up_bias"] = 0.1 * rand(N), 0.1 * rand(N)
    return s


_INPUTS = {"embed": _embed_inputs, "layernorm": _norm_inputs, "gated": _gated_inputs}


def _outputs(case):
    """Names, shapes and types of what a pass writes."""
    M, x, y, grad = case["M"], case["x"], case["y"], case["dir"] == "grad"
    if case["op"] == "embed":
        if grad:
            return {} if case["accumulate"] else {"dtable": ((case["V"], case["C"]), x)}
        return {"y": ((M, case["C"]), y)}
    if case["op"] == "layernorm":
        C = case["C"]
        if grad:
            return {"dx": ((M, C), x), "dweight": ((C,), "f32"), "dbias": ((C,), "f32")}
        out = {"y": ((M, C), y), "mean": ((M,), "f32"), "rstd": ((M,), "f32")}
        if y == "fp8":
            out["y_scale"] = ((M,), "f32")
        if case["residual"]:
            out["sum"] = ((M, C), x)
        return out
    K, N = case["K"], case["N"]
    if grad:
        out = {"dx": ((M, K), x), "dw_gate": ((N, K), x), "dw_up": ((N, K), x)}
        if case["bias"]:
            out["dgate_bias"], out["dup_bias"] = ((N,), "f32"), ((N,), "f32")
        return out
    out = {"y": ((M, N), y)}
    if case["save"]:
        out["z_gate"], out["z_up"] = ((M, N), y), ((M, N), y)
    return out


def prepare(case, seed):
    s = dict(case=case)
    s["in"] = _INPUTS[case["op"]](case, seed)
    s["out"] = {k: torch.empty(shape, dtype=_TORCH[kind], device="cuda")
                for k, (shape, kind) in _outputs(case).items()}
    s["buf"] = {k: _Buf(v) for k, v in {**s["in"], **s["out"]}.items()}
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


def _plain_embed(case, i):
    ids, V = i["ids"].long(), case["V"]
    inside = (ids >= 0) & (ids < V)
    if case["dir"] == "forward":
        at = ids.clamp(0, V - 1)
        y = i["table"][at].float() * _scale(case)
        if case["x"] == "fp8":
            y = y * i["table_scale"][at][:, None]
        y = torch.where(inside[:, None], y, torch.zeros_like(y))
        return dict(y=y.to(_TORCH[case["y"]]))
    # A row more takes what is outside.
    d = torch.zeros((V + 1, case["C"]), device="cuda")
    d.index_add_(0, torch.where(inside, ids, torch.full_like(ids, V)), i["dy"].float())
    d = d[:V] * _scale(case)
    if case["accumulate"]:
        i["dtable"].copy_(i["dtable"].float() + d)
        return dict(dtable=i["dtable"])
    return dict(dtable=d.to(_TORCH[case["x"]]))


def _plain_norm(case, i):
    if case["dir"] == "grad":
        # x is the saved sum here; the residual's case has its gradient too.
        x, dy, r = i["x"].float(), i["dy"].float(), i["rstd"][:, None]
        h, g = (x - i["mean"][:, None]) * r, dy * i["weight"]
        dx = r * (g - g.mean(dim=1, keepdim=True) - h * (g * h).mean(dim=1, keepdim=True))
        if case["residual"]:
            dx = dx + i["residual"].float()
        return dict(dx=dx.to(i["x"].dtype), dweight=(dy * h).sum(dim=0), dbias=dy.sum(dim=0))
    t = i["x"].float()
    if case["residual"]:
        t = t + i["residual"].float()
    mean = t.mean(dim=1)
    centred = t - mean[:, None]
    rstd = torch.rsqrt(centred.square().mean(dim=1) + _EPS)
    y = centred * rstd[:, None] * i["weight"] + i["bias"]
    out = dict(mean=mean, rstd=rstd)
    if case["residual"]:
        out["sum"] = t.to(i["x"].dtype)
    if case["y"] == "fp8":
        out["y"], out["y_scale"] = _to_fp8(y)
    else:
        out["y"] = y.to(_TORCH[case["y"]])
    return out


def _plain_gated(case, i):
    x, wg, wu = i["x"].float(), i["w_gate"].float(), i["w_up"].float()
    if case["x"] == "fp8":
        x = x * i["x_scale"][:, None]
        wg, wu = wg * i["gate_scale"][:, None], wu * i["up_scale"][:, None]
    if case["dir"] == "grad":
        zg, zu, dy = i["z_gate"].float(), i["z_up"].float(), i["dy"].float()
        dg, du = dy * zu * _act_grad(zg, case["act"]), dy * _act(zg, case["act"])
        xt = i["x"].dtype
        out = dict(dx=(torch.matmul(dg, wg) + torch.matmul(du, wu)).to(xt),
                   dw_gate=torch.matmul(dg.t(), x).to(xt), dw_up=torch.matmul(du.t(), x).to(xt))
        if case["bias"]:
            out["dgate_bias"], out["dup_bias"] = dg.sum(dim=0), du.sum(dim=0)
        return out
    zg, zu = torch.matmul(x, wg.t()), torch.matmul(x, wu.t())
    if case["bias"]:
        zg, zu = zg + i["gate_bias"], zu + i["up_bias"]
    yt = _TORCH[case["y"]]
    out = dict(y=(_act(zg, case["act"]) * zu).to(yt))
    if case["save"]:
        out["z_gate"], out["z_up"] = zg.to(yt), zu.to(yt)
    return out


_PLAIN = {"embed": _plain_embed, "layernorm": _plain_norm, "gated": _plain_gated}


# ------------------------------------------------------------------- passes
def _own(s):
    vs, case, b = _package(), s["case"], s["buf"]
    get = b.get
    if case["op"] == "embed":
        if case["dir"] == "forward":
            vs.run_embed_gpu(b["table"], b["ids"], b["y"], scale=_scale(case),
                             table_scale=get("table_scale"))
            return s["out"]
        vs.run_embed_grad_gpu(b["dy"], b["ids"], b["dtable"], scale=_scale(case),
                              accumulate=case["accumulate"])
        return dict(dtable=b["dtable"].t)
    if case["op"] == "layernorm":
        if case["dir"] == "forward":
            vs.run_layernorm_gpu(b["x"], b["weight"], b["y"], bias=b["bias"],
                                 residual=get("residual"), sum=get("sum"), y_scale=get("y_scale"),
                                 mean=b["mean"], rstd=b["rstd"], eps=_EPS)
        else:
            vs.run_layernorm_grad_gpu(b["dy"], b["x"], b["weight"], b["mean"], b["rstd"], b["dx"],
                                      b["dweight"], b["dbias"], dsum=get("residual"))
    elif case["dir"] == "forward":
        vs.run_gated_gpu(b["x"], b["w_gate"], b["w_up"], b["y"], gate_bias=get("gate_bias"),
                         up_bias=get("up_bias"), act=case["act"], z_gate=get("z_gate"),
                         z_up=get("z_up"), x_scale=get("x_scale"), gate_scale=get("gate_scale"),
                         up_scale=get("up_scale"))
    else:
        vs.run_gated_grad_gpu(b["dy"], b["x"], b["w_gate"], b["w_up"], b["z_gate"], b["z_up"],
                              act=case["act"], dx=b["dx"], dw_gate=b["dw_gate"],
                              dw_up=b["dw_up"], dgate_bias=get("dgate_bias"),
                              dup_bias=get("dup_bias"))
    return s["out"]


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["case"]["op"]](state["case"], state["in"])


def _rows_met(case):
    """Table rows that the tokens of a pass are expected to meet."""
    M, V = case["M"], case["V"]
    k = np.arange(1, V + 1, dtype=np.float64)
    p = np.log1p(1 / k) / math.log(V + 1) * (31 / 32)
    return float(np.sum(-np.expm1(M * np.log1p(-p))))


def work(case):
    M, xs, ys = case["M"], _SIZE[case["x"]], _SIZE[case["y"]]
    grad = case["dir"] == "grad"
    if case["op"] == "embed":
        C = case["C"]
        if not grad:
            row = C * xs + (4 if case["x"] == "fp8" else 0)
            return {"bytes": _rows_met(case) * row + M * (C * ys + 4.0), "flops": float(M * C)}
        table = 2 * _rows_met(case) if case["accumulate"] else case["V"]
        return {"bytes": table * C * xs + M * (C * ys + 4.0), "flops": float(M * C)}
    if case["op"] == "layernorm":
        C, r = case["C"], case["residual"]
        if not grad:
            each = xs * (3 if r else 1) + ys
            rows = 8 + (4 if case["y"] == "fp8" else 0)
        else:
            each, rows = xs * (3 if r else 2) + ys, 8
        return {"bytes": float(M * C * each + M * rows + C * (12 if grad else 8)),
                "flops": 10.0 * M * C}
    K, N = case["K"], case["N"]
    bias = 8 * N if case["bias"] else 0
    if not grad:
        return {"bytes": float((M + 2 * N) * K * xs + M * N * ys * (3 if case["save"] else 1) + bias
                               + (4 * (M + 2 * N) if case["x"] == "fp8" else 0)),
                "flops": 4.0 * M * N * K}
    return {"bytes": float(2 * (M + 2 * N) * K * xs + 3 * M * N * ys + bias),
            "flops": 8.0 * M * N * K}


# ------------------------------------------------------------------ 64 bits
def _exact_embed(case, i):
    ids, V, C = i["ids"].long(), case["V"], case["C"]
    kept = torch.nonzero((ids >= 0) & (ids < V)).view(-1)
    if case["dir"] == "forward":
        y = torch.zeros((case["M"], C), dtype=torch.float64, device="cuda")
        rows = i["table"][ids[kept]].to(torch.float32).double()
        if case["x"] == "fp8":
            rows = rows * i["table_scale"][ids[kept]].double().unsqueeze(1)
        y[kept] = rows * math.sqrt(C)
        return dict(y=y)
    d = torch.zeros((V, C), dtype=torch.float64, device="cuda")
    d.index_put_((ids[kept],), i["dy"][kept].double() * math.sqrt(C), accumulate=True)
    return dict(dtable=d + i["dtable"].double() if case["accumulate"] else d)


def _exact_norm(case, i):
    x, w = i["x"].double(), i["weight"].double()
    C = x.shape[1]
    if case["dir"] == "grad":
        dy, r, mu = (i[k].double() for k in ("dy", "rstd", "mean"))
        r, c = r.unsqueeze(1), x - mu.unsqueeze(1)
        # The Jacobian of s -> (s - mean(s)) * rstd(s), applied row by row.
        v = dy * w
        dx = r * v - r * v.sum(1, keepdim=True) / C - r.pow(3) * c * torch.sum(v * c, 1, keepdim=True) / C
        if case["residual"]:
            dx = dx + i["residual"].double()
        return dict(dx=dx, dweight=torch.sum(dy * c * r, 0), dbias=torch.sum(dy, 0))
    if case["residual"]:
        x = x + i["residual"].double()
    mu = torch.sum(x, 1) / C
    sd = torch.sqrt(torch.sum((x - mu.unsqueeze(1)) ** 2, 1) / C + _EPS)
    y = w * (x - mu.unsqueeze(1)) / sd.unsqueeze(1) + i["bias"].double()
    out = dict(mean=mu, rstd=1 / sd)
    if case["residual"]:
        out["sum"] = x
    if case["y"] == "fp8":
        out["y_scale"] = torch.clamp(y.abs().max(1).values, min=_TINY) / _FP8_MAX
        y = y / out["y_scale"].unsqueeze(1)
    out["y"] = y
    return out


def _exact_gated(case, i):
    x, wg, wu = (i[k].to(torch.float32).double() for k in ("x", "w_gate", "w_up"))
    if case["x"] == "fp8":
        x = x * i["x_scale"].double().view(-1, 1)
        wg, wu = wg * i["gate_scale"].double().view(-1, 1), wu * i["up_scale"].double().view(-1, 1)

    def act(z):
        if case["act"] == "relu":
            return torch.where(z > 0, z, torch.zeros_like(z))
        if case["act"] == "gelu":
            # 0.5 (1 + tanh u) is the logistic function of 2u.
            return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
        return z * torch.sigmoid(z) if case["act"] == "silu" else z

    if case["dir"] == "forward":
        zg, zu = x @ wg.T, x @ wu.T
        if case["bias"]:
            zg, zu = zg + i["gate_bias"].double(), zu + i["up_bias"].double()
        out = dict(y=act(zg) * zu)
        if case["save"]:
            out["z_gate"], out["z_up"] = zg, zu
        return out
    zg, zu = (i[k].double().requires_grad_(True) for k in ("z_gate", "z_up"))
    with torch.enable_grad():
        dg, du = torch.autograd.grad(act(zg) * zu, (zg, zu), i["dy"].double())
    out = dict(dx=dg @ wg + du @ wu, dw_gate=dg.T.contiguous() @ x, dw_up=du.T.contiguous() @ x)
    if case["bias"]:
        out["dgate_bias"], out["dup_bias"] = dg.sum(0), du.sum(0)
    return out


def exact(case, seed):
    form = {"embed": _exact_embed, "layernorm": _exact_norm, "gated": _exact_gated}[case["op"]]
    return form(case, _INPUTS[case["op"]](case, seed))
