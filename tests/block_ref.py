"""64-bit formulas and tolerances for the tests of layer norm, the embedding and the
gated projection.  u = 2^-24 (EPS) is half an ulp of FP32 at 1."""
from __future__ import annotations

import numpy as np

from dense_ref import EPS, ROUND, TINY, act, act_grad, pack, unpack


def values(rng, shape, kind, scale=1.0):
    """Random values that `kind` holds exactly."""
    return unpack(pack(scale * rng.standard_normal(shape), kind), kind)


def rounding(v, kind):
    return np.abs(v) * ROUND[kind] + TINY[kind]


# ------------------------------------------------------------------ layer norm
def layer_norm(x, r, w, b, eps):
    """(t, mean, rstd, y) by rows."""
    t = x if r is None else x + r
    mean = np.mean(t, axis=1, keepdims=True)
    rstd = 1 / np.sqrt(np.mean((t - mean) ** 2, axis=1, keepdims=True) + eps)
    return t, mean, rstd, (t - mean) * rstd * w + (0 if b is None else b)


def layer_norm_tol(t, mean, rstd, w, b, eps):
    """Errors of (mean, rstd, y) in FP32.  A row's sum is added in chains of at most
    L = C / 8 + 16 terms, so mean is off by em = (L + 2) u mean|t|; d = t - mean by ed =
    em + u (|t| + |d|).  em is common to the row and the d's sum is zero, so the variance
    gets em^2, the roundings of each d twice, and its own chain."""
    C = t.shape[1]
    L = C / 8 + 16
    d = np.abs(t - mean)
    em = (L + 2) * EPS * np.mean(np.abs(t), axis=1, keepdims=True)
    own = EPS * (np.abs(t) + d)
    var = np.mean(d * d, axis=1, keepdims=True)
    rv = (2.2 * np.mean(d * own, axis=1, keepdims=True) + em ** 2 +
          np.mean(own ** 2, axis=1, keepdims=True) + (L + 4) * EPS * var) * rstd ** 2
    # 1 / sqrt(1 + r): r / 2, and no more than 0.6 r for r under 0.1.
    rr = 0.6 * rv + 4 * EPS
    y = np.abs(w) * rstd * (em + own + d * rr) + 4 * EPS * (np.abs(w) * d * rstd +
                                                            (0 if b is None else np.abs(b)))
    return em + EPS * np.abs(mean), rstd * rr, y


def layer_norm_grad(dy, s, w, mean, rstd, dsum):
    """(dx, dweight, dbias), and their errors in FP32: chains of a row's C values for the
    two sums and of the M rows for the other two."""
    M, C = s.shape
    h, g = (s - mean) * rstd, dy * w
    mg, mgh = np.mean(g, axis=1, keepdims=True), np.mean(g * h, axis=1, keepdims=True)
    dx = rstd * (g - mg - h * mgh) + (0 if dsum is None else dsum)
    ah, ag = np.abs(h), np.abs(g)
    sg, sgh = np.mean(ag, axis=1, keepdims=True), np.mean(ag * ah, axis=1, keepdims=True)
    tol = rstd * ((C + 6) * EPS * (sg + ah * sgh) + 8 * EPS * (ag + sg + ah * sgh)) + \
        8 * EPS * np.abs(dx)
    tw = (M + 8) * EPS * np.sum(np.abs(dy) * ah, axis=0) + 1e-30
    tb = (M + 4) * EPS * np.sum(np.abs(dy), axis=0) + 1e-30
    return (dx, np.sum(dy * h, axis=0), np.sum(dy, axis=0)), (tol, tw, tb)


# ------------------------------------------------------------ gated projection
def gated(x, wg, wu, bg, bu, kind):
    """(z_gate, z_up, y) and their errors in FP32: sums of K products and a bias in any
    order; each act's slope is at most 1.13, and its own arithmetic good to 16 u."""
    K = x.shape[1]
    out, tol = [], []
    for w, b in ((wg, bg), (wu, bu)):
        out.append(x @ w.T + (0 if b is None else b))
        tol.append((K + 4) * EPS * (np.abs(x) @ np.abs(w).T + (0 if b is None else np.abs(b))))
    a = act(out[0], kind)
    ta = 1.13 * tol[0] + 16 * EPS * np.abs(out[0])
    y = a * out[1]
    ty = (np.abs(a) + ta) * tol[1] + np.abs(out[1]) * ta + 2 * EPS * np.abs(y)
    return (*out, y), (*tol, ty)


def gated_grad(dy, x, wg, wu, zg, zu, kind, operand):
    """dx, dw_gate, dw_up, dgate_bias, dup_bias and their errors: act' is at most 1.13
    and good to 32 u there, act to 16 u |z|, two products each; both dz round to the
    operands' type; sums of 2 N and of M products in any order."""
    M, N = dy.shape
    dg, du = dy * zu * act_grad(zg, kind), dy * act(zg, kind)
    eg, eu = 44 * EPS * 1.13 * np.abs(dy * zu), 20 * EPS * np.abs(dy * zg)
    bias = (dg.sum(0), du.sum(0))
    tb = (eg.sum(0) + (M + 4) * EPS * np.abs(dg).sum(0), eu.sum(0) + (M + 4) * EPS * np.abs(du).sum(0))
    if operand == "bf16":
        eg, eu = eg + rounding(dg, "bf16") * 1.01, eu + rounding(du, "bf16") * 1.01
    ag, au = np.abs(dg), np.abs(du)
    dx = dg @ wg + du @ wu
    tx = eg @ np.abs(wg) + eu @ np.abs(wu) + (2 * N + 6) * EPS * (ag @ np.abs(wg) + au @ np.abs(wu))
    tg = eg.T @ np.abs(x) + (M + 4) * EPS * (ag.T @ np.abs(x))
    tu = eu.T @ np.abs(x) + (M + 4) * EPS * (au.T @ np.abs(x))
    return (dx, dg.T @ x, du.T @ x, *bias), (tx, tg, tu, *tb)
