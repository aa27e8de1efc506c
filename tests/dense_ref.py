"""Value types, 64-bit formulas and device helpers for the tests of the dense
operators (RMS norm, linear, AdamW)."""
from __future__ import annotations

import numpy as np

EPS = 2.0 ** -24  # half an ulp of FP32 at 1
ROUND = {"f32": EPS, "bf16": 2.0 ** -8}  # relative error of one rounding (8 significant bits)
TINY = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133}  # smallest magnitudes


def to_bf16(a):
    """float -> bf16 bit patterns, nearest even; NaN stays NaN."""
    a = np.ascontiguousarray(a, np.float32)
    u = a.view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(a), np.uint16(0x7FC0), r)


def from_bf16(u):
    return (u.astype(np.uint32) << 16).view(np.float32)


def _e4m3_table():
    t = np.zeros(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        t[c] = np.nan if (c & 127) == 127 else (-v if c & 128 else v)
    return t


E4M3 = _e4m3_table()


def from_fp8(u):
    return E4M3[u]


def to_fp8(a):
    """float -> e4m3 codes, nearest (ties to the even code), |a| <= 448."""
    a = np.asarray(a, np.float64)
    pos = E4M3[:127]
    mag = np.abs(a)
    hi = np.clip(np.searchsorted(pos, mag), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = mag - pos[lo], pos[hi] - mag
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi).astype(np.uint8)
    return code | np.where(np.signbit(a), np.uint8(128), np.uint8(0))


def pack(a, kind):
    return {"f32": lambda: np.ascontiguousarray(a, np.float32), "bf16": lambda: to_bf16(a),
            "fp8": lambda: to_fp8(a)}[kind]()


def unpack(u, kind):
    """Bit patterns (or float32) -> float64 values."""
    return {"f32": lambda: u.astype(np.float64),
            "bf16": lambda: from_bf16(u).astype(np.float64), "fp8": lambda: from_fp8(u)}[kind]()


NP = {"f32": np.float32, "bf16": np.uint16, "fp8": np.uint8}
_GUARD = {"f32": np.float32(-7.25e11), "bf16": np.uint16(0xD37C), "fp8": np.uint8(0x5B)}


class Mat:
    """A device matrix of `rows` x `cols` values with a row stride and a first
    element off the allocation's start, in a buffer filled with a guard value
    that nothing but the matrix's own elements may change."""

    def __init__(self, vs, st, values, kind, pad=0, off=0, shape=None):
        rows, cols = shape if values is None else values.shape
        self.vs, self.st, self.kind, self.rows, self.cols = vs, st, kind, rows, cols
        self.ld, self.off = cols + pad, off
        self.host = np.full(off + rows * self.ld + 64, _GUARD[kind], NP[kind])
        if values is not None and rows:
            self.grid(self.host)[:, :cols] = pack(values, kind)
        self.buf = vs.DeviceArray.from_numpy(self.host, st)
        size = self.host.itemsize
        self.view = vs.DeviceView(self.buf.ptr.value + off * size, (rows, cols), NP[kind],
                                  ld=self.ld, owner=self.buf)

    def grid(self, flat):
        return flat[self.off:self.off + self.rows * self.ld].reshape(self.rows, self.ld)

    def codes(self):
        """The matrix's bit patterns; checks that the guard is whole."""
        flat = self.buf.numpy(self.st)
        g = self.grid(flat)[:, :self.cols].copy()
        self.grid(flat)[:, :self.cols] = self.grid(self.host)[:, :self.cols]
        assert flat.tobytes() == self.host.tobytes(), "written outside the matrix"
        return g

    def values(self):
        return unpack(self.codes(), self.kind)


def vector(vs, st, a):
    return vs.DeviceArray.from_numpy(np.ascontiguousarray(a, np.float32), st)


# ---------------------------------------------------------------- formulas
def rms_norm(x, r, w, eps):
    t = x if r is None else x + r
    rstd = 1 / np.sqrt(np.mean(t * t, axis=1, keepdims=True) + eps)
    return t, rstd, t * rstd * w


def rms_norm_grad(dy, s, w, rstd, dsum):
    h = s * rstd
    g = dy * w
    dx = rstd * (g - h * np.mean(g * h, axis=1, keepdims=True))
    return dx + (0 if dsum is None else dsum), (dy * h).sum(0)


def act(z, kind):
    if kind == "relu":
        return np.where(z < 0, 0, z)
    if kind == "gelu":
        return 0.5 * z * (1 + np.tanh(np.sqrt(2 / np.pi) * (z + 0.044715 * z ** 3)))
    if kind == "silu":
        return z / (1 + np.exp(-z))
    return z


def act_grad(z, kind):
    if kind == "relu":
        return (z > 0).astype(np.float64)
    if kind == "gelu":
        t = np.tanh(np.sqrt(2 / np.pi) * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * np.sqrt(2 / np.pi) * (1 + 0.134145 * z ** 2)
    if kind == "silu":
        p = 1 / (1 + np.exp(-z))
        return p * (1 + z * (1 - p))
    return np.ones_like(z)


def close(got, want, tol, what):
    """Every element within its tolerance; NaN and infinities in the same places."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    tol = np.broadcast_to(tol, want.shape)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    odd = ~np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN elsewhere"
    assert np.array_equal(got[odd & ~np.isnan(want)], want[odd & ~np.isnan(want)]), what
    err = np.where(odd, 0, np.abs(np.where(odd, 0, got) - np.where(odd, 0, want)))
    if err.size:
        at = np.unravel_index(np.argmax(err - np.where(odd, np.inf, tol)), err.shape)
        assert odd[at] or err[at] <= tol[at], \
            f"{what}: {got[at]!r} for {want[at]!r} at {at}, error {err[at]:.3e} over {tol[at]:.3e}"
