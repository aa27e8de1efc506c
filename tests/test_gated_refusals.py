"""Arguments the gated projection and its gradient refuse, before any device work, and
which kernels its sizes take (CPU)."""
from __future__ import annotations

import ctypes as C

import pytest

from dense_plans import TILES
from gated_plans import forced, gated_grad_plan, gated_plan
from test_dense_refusals import bf, f8, mat, refused
from test_gpu_gated import GATED_SIZES

P = [1 << 20 << i for i in range(12)]

FORWARD = {
    "w_up of another shape": dict(w_up=mat(6, 8, ptr=P[2])),
    "w_up of another type": dict(w_up=bf(5, 8, ptr=P[2])),
    "w_gate of another length": dict(w_gate=mat(5, 9, ptr=P[1])),
    "y of another shape": dict(y=mat(4, 6, ptr=P[3])),
    "8-bit y": dict(y=f8(4, 5, ptr=P[3])),
    "8-bit without scales": dict(x=f8(4, 8), w_gate=f8(5, 8), w_up=f8(5, 8)),
    "8-bit with two scales": dict(x=f8(4, 8), w_gate=f8(5, 8, ptr=P[1]), w_up=f8(5, 8, ptr=P[2]),
                                  x_scale=mat(4), gate_scale=mat(5)),
    "scales without 8-bit": dict(x_scale=mat(4), gate_scale=mat(5), up_scale=mat(5)),
    "short up_scale": dict(x=f8(4, 8), w_gate=f8(5, 8), w_up=f8(5, 8), x_scale=mat(4),
                           gate_scale=mat(5), up_scale=mat(4)),
    "short gate_bias": dict(gate_bias=mat(4)),
    "misaligned up_bias": dict(up_bias=mat(5, ptr=4098)),
    "unknown activation": dict(act="tanh"),
    "z_gate alone": dict(z_gate=mat(4, 5, ptr=P[4])),
    "z_up alone": dict(z_up=mat(4, 5, ptr=P[4])),
    "z of another type": dict(z_gate=bf(4, 5, ptr=P[4]), z_up=bf(4, 5, ptr=P[5])),
    "z of two strides": dict(z_gate=mat(4, 5, ptr=P[4], ld=8), z_up=mat(4, 5, ptr=P[5])),
    "z_gate over z_up": dict(z_gate=mat(4, 5, ptr=P[4]), z_up=mat(4, 5, ptr=P[4])),
    "z_up over y": dict(z_gate=mat(4, 5, ptr=P[4]), z_up=mat(4, 5, ptr=P[3])),
    "y over x": dict(x=mat(5, 5, ptr=P[3]), w_gate=mat(5, 5, ptr=P[1]), w_up=mat(5, 5, ptr=P[2]),
                     y=mat(5, 5, ptr=P[3])),
    "y over w_up": dict(w_up=mat(5, 8, ptr=P[3])),
    "z_gate over w_gate": dict(z_gate=mat(4, 5, ptr=P[1]), z_up=mat(4, 5, ptr=P[5])),
    "misaligned w_up": dict(w_up=mat(5, 8, ptr=P[2] + 1)),
    "no w_up": dict(w_up=mat(5, 8, ptr=0)),
    "short workspace": dict(x=mat(64, 8192), w_gate=mat(5, 8192, ptr=P[1]),
                            w_up=mat(5, 8192, ptr=P[2]), y=mat(64, 5, ptr=P[3]), workspace=f8(16)),
}


@pytest.mark.parametrize("case", FORWARD)
def test_gated_refuses(vs, case):
    kw = dict(x=mat(4, 8), w_gate=mat(5, 8, ptr=P[1]), w_up=mat(5, 8, ptr=P[2]),
              y=mat(4, 5, ptr=P[3]))
    kw.update(FORWARD[case])
    refused(vs, vs.VCSR_EINVAL, vs.run_gated_gpu, **kw)


def operands():
    return dict(dy=mat(8, 8, ptr=P[0]), x=mat(8, 8, ptr=P[1]), w_gate=mat(8, 8, ptr=P[2]),
                w_up=mat(8, 8, ptr=P[3]), z_gate=mat(8, 8, ptr=P[4]), z_up=mat(8, 8, ptr=P[5]))


OUT = dict(dx=mat(8, 8, ptr=P[6]), dw_gate=mat(8, 8, ptr=P[7]), dw_up=mat(8, 8, ptr=P[8]))
GRAD = {
    "no z_gate": dict(z_gate=None, dx=OUT["dx"]),
    "no z_up": dict(z_up=None, dx=OUT["dx"], act="none"),
    "z of another type": dict(z_up=bf(8, 8), dx=OUT["dx"]),
    "z of two strides": dict(z_up=mat(8, 8, ld=9), dx=OUT["dx"]),
    "8-bit operands": dict(x=f8(8, 8), w_gate=f8(8, 8), w_up=f8(8, 8), dx=f8(8, 8)),
    "8-bit dy": dict(dy=f8(8, 8), z_gate=f8(8, 8), z_up=f8(8, 8), dx=OUT["dx"]),
    "dx of another type": dict(dx=bf(8, 8, ptr=P[6])),
    "dw of another shape": dict(dw_gate=mat(8, 7), dw_up=OUT["dw_up"]),
    "dw_gate alone": dict(dw_gate=OUT["dw_gate"]),
    "dw_up alone": dict(dw_up=OUT["dw_up"]),
    "dw_gate over dw_up": dict(dw_gate=OUT["dw_up"], dw_up=OUT["dw_up"]),
    "short dgate_bias": dict(dgate_bias=mat(7)),
    "misaligned dup_bias": dict(dup_bias=mat(8, ptr=4098)),
    "dgate_bias over dup_bias": dict(dgate_bias=mat(8), dup_bias=mat(8)),
    "dx over w_gate": dict(dx=mat(8, 8, ptr=P[2])),
    "dx over w_up": dict(dx=mat(8, 8, ptr=P[3])),
    "dx over x, with dw": dict(OUT, dx=mat(8, 8, ptr=P[1])),
    "dx over dw_up": dict(OUT, dx=OUT["dw_up"]),
    "dw_gate over x": dict(OUT, dx=None, dw_gate=mat(8, 8, ptr=P[1])),
    "dw_up over w_up, with dx": dict(OUT, dw_up=mat(8, 8, ptr=P[3])),
    "dw_up over w_gate, with dx": dict(OUT, dw_up=mat(8, 8, ptr=P[2])),
    "short workspace": dict(OUT, workspace=f8(64)),
    "misaligned workspace": dict(OUT, workspace=f8(1 << 20, ptr=4104)),
    "no workspace": dict(OUT, workspace=f8(1 << 20, ptr=0)),
}


@pytest.mark.parametrize("case", GRAD)
def test_gated_grad_refuses(vs, case):
    kw = dict(operands(), workspace=mat(1 << 20, ptr=1 << 36))
    kw.update(GRAD[case])
    refused(vs, vs.VCSR_EINVAL, vs.run_gated_grad_gpu, **kw)


def test_gated_sizes_past_the_kernels_are_a_range_error(vs):
    lib, need = vs.load_library(), C.c_size_t(0)
    ok = dict(M=4, N=4, K=4, x=P[0], w_gate=P[1], w_up=P[2], y=P[3])
    for bad in (dict(M=1 << 31), dict(N=(1 << 29) + 1), dict(K=(1 << 20) + 1),
                dict(ldwu=(1 << 20) + 1), dict(M=(1 << 31) - 1, N=1 << 20)):
        a = vs._GatedArgs(**{**ok, **bad})
        assert lib.vcsr_gated(C.byref(a), None, None) == vs.VCSR_ERANGE, bad
    ok = dict(M=4, N=4, K=4, dy=P[0], z_gate=P[1], z_up=P[2], x=P[3], w_gate=P[4], w_up=P[5],
              dx=P[6])
    for bad in (dict(M=1 << 31), dict(N=(1 << 20) + 1), dict(K=(1 << 20) + 1),
                dict(ldwg=(1 << 20) + 1), dict(M=(1 << 31) - 1, K=1 << 20)):
        a = vs._GatedGradArgs(**{**ok, **bad})
        assert lib.vcsr_gated_grad(C.byref(a), None, None) == vs.VCSR_ERANGE, bad
    for fn in ("vcsr_gated", "vcsr_gated_grad"):
        assert getattr(lib, fn)(None, None, None) == vs.VCSR_EINVAL, fn
    for fn in ("vcsr_gated_workspace", "vcsr_gated_grad_workspace"):
        assert getattr(lib, fn)(None, C.byref(need)) == vs.VCSR_EINVAL, fn
        assert getattr(lib, fn)(None, None) == vs.VCSR_EINVAL, fn
    a = vs._GatedArgs(M=4, N=4, K=4, z_gate=16)
    assert lib.vcsr_gated_workspace(C.byref(a), C.byref(need)) == vs.VCSR_OK


def test_gated_without_a_gpu_says_so(vs):
    if vs.device_count() > 0:
        pytest.skip("a GPU is visible")
    refused(vs, vs.VCSR_EDEVICE, vs.run_gated_gpu, mat(4, 8), mat(5, 8, ptr=P[1]),
            mat(5, 8, ptr=P[2]), mat(4, 5, ptr=P[3]))
    for over in (dict(OUT), dict(dx=mat(8, 8, ptr=P[1])), dict(dx=mat(8, 8, ptr=P[0])),
                 dict(dw_gate=mat(8, 8, ptr=P[2]), dw_up=mat(8, 8, ptr=P[3]))):
        refused(vs, vs.VCSR_EDEVICE, vs.run_gated_grad_gpu, **operands(), **over,
                workspace=mat(1 << 20, ptr=1 << 36))


@pytest.mark.parametrize("size", GATED_SIZES, ids=lambda s: "x".join(map(str, s[:4])))
def test_gated_forward_sizes(vs, size):
    got = gated_plan(vs, *size[:4])
    assert all(w is None or g == w for g, w in zip(got, size[4])), got


def test_gated_forced_plans(vs):
    free = gated_plan(vs, 300, 300, 700, "bf16")
    for kind, tiles in TILES.items():
        for tile, stages in tiles:
            with forced(vs, tile, stages, splits=2):
                assert gated_plan(vs, 300, 300, 700, kind) == (tile, stages, 2, 300)
            with forced(vs, tile, stages, rows=tile):
                assert gated_plan(vs, 300, 300, 700, kind) == (tile, stages, 1, tile)
    with forced(vs, 256, together=True):
        assert gated_grad_plan(vs, 300, 300, 700, "bf16") == (1, 256, 1, 256, 1)
    with forced(vs, 128, splits=3):
        assert gated_grad_plan(vs, 300, 300, 700, "f32") == (0, 128, 3, 128, 3)
    assert gated_plan(vs, 300, 300, 700, "bf16") == free
