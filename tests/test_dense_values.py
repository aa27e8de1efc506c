"""Host conversions of the binding's value types (CPU)."""
from __future__ import annotations

import numpy as np

from dense_ref import E4M3, from_bf16, to_bf16, to_fp8


def test_bf16_conversions(vs):
    rng = np.random.default_rng(0)
    a = np.concatenate([rng.standard_normal(1000) * 2.0 ** rng.integers(-120, 120, 1000),
                        [0.0, -0.0, np.inf, -np.inf, 1.00390625, 1.01171875, 3.3895314e38]])
    a = a.astype(np.float32)
    assert np.array_equal(vs.to_bf16(a), to_bf16(a))
    assert np.array_equal(vs.from_bf16(vs.to_bf16(a)), from_bf16(to_bf16(a)))
    assert np.isnan(vs.from_bf16(vs.to_bf16(np.float32([np.nan])))).all()


def test_e4m3_codes_are_their_own_values(vs):
    codes = np.arange(256, dtype=np.uint8)
    assert np.array_equal(vs.from_fp8(codes), E4M3.astype(np.float32), equal_nan=True)
    # A row whose largest value is 448 has scale 1 and comes back code for code.
    row = E4M3[[c for c in range(256) if c & 127 != 127]][None, :].astype(np.float32)
    got, scale = vs.quantize_fp8(row)
    assert scale[0] == 1.0 and np.array_equal(vs.from_fp8(got), row)


def test_quantize_rounds_to_the_nearest_code(vs):
    rng = np.random.default_rng(1)
    a = (rng.standard_normal((20, 300)) * 2.0 ** rng.integers(-12, 3, (20, 300))).astype(np.float32)
    a[3] = 0
    a[4, 0] = 448
    a[4, 1:4] = [1.0625, 1.1875, 2.0 ** -10]  # halfway: to the even code
    codes, scale = vs.quantize_fp8(a)
    want = np.maximum(np.abs(a).max(1), np.float32(1e-30)) / np.float32(448)
    assert np.array_equal(scale, want.astype(np.float32))
    ref = to_fp8(np.clip(a / scale[:, None], -448, 448))
    assert np.array_equal(vs.from_fp8(codes), vs.from_fp8(ref))
    assert not vs.from_fp8(codes[3]).any()


def test_device_view_describes_a_strided_matrix(vs):
    v = vs.DeviceView(4096, (5, 7), vs.BF16, ld=16)
    assert v.nbytes == (4 * 16 + 7) * 2 and v.ld == 16 and v.ptr.value == 4096
    assert vs.DeviceView(0, (0, 7), vs.F32).nbytes == 0
