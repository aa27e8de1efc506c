"""Arguments the embedding and its gradient refuse, before any device work (CPU)."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from test_dense_refusals import Fake, bf, f8, mat, refused


def ids(n, **kw):
    return Fake((n,), np.int32, **kw)


FORWARD = {
    "ids of 64 bits": dict(ids=Fake((4,), np.int64)),
    "ids of float32": dict(ids=mat(4)),
    "a matrix of ids": dict(ids=Fake((4, 1), np.int32)),
    "short ids": dict(ids=ids(4, nbytes=12)),
    "no ids": dict(ids=ids(4, ptr=0)),
    "misaligned ids": dict(ids=ids(4, ptr=4098)),
    "y of another shape": dict(y=mat(4, 7)),
    "y for other tokens": dict(y=mat(5, 8)),
    "8-bit y": dict(y=f8(4, 8)),
    "8-bit table without scales": dict(table=f8(9, 8)),
    "scales without 8-bit table": dict(table_scale=mat(9)),
    "short scales": dict(table=f8(9, 8), table_scale=mat(8)),
    "table of no known type": dict(table=Fake((9, 8), np.int32)),
    "no table": dict(table=mat(9, 8, ptr=0)),
    "no y": dict(y=mat(4, 8, ptr=0)),
    "misaligned table": dict(table=mat(9, 8, ptr=4098)),
    "table too short for its stride": dict(table=mat(9, 8, ld=64, nbytes=128)),
    "stride under the row": dict(table=mat(9, 8, ld=6, nbytes=4096)),
    "y over the table": dict(table=mat(4, 8, ptr=8192), y=mat(4, 8, ptr=8192)),
    "scale not finite": dict(scale=float("nan")),
    "an empty table": dict(table=mat(0, 8)),
    "no columns": dict(table=mat(9, 0), y=mat(4, 0)),
}


@pytest.mark.parametrize("case", FORWARD)
def test_embed_refuses(vs, case):
    kw = dict(table=mat(9, 8), ids=ids(4), y=mat(4, 8, ptr=65536))
    kw.update(FORWARD[case])
    refused(vs, vs.VCSR_EINVAL, vs.run_embed_gpu, **kw)


GRAD = {
    "ids of 64 bits": dict(ids=Fake((4,), np.int64)),
    "short ids": dict(ids=ids(4, nbytes=12)),
    "dy of another shape": dict(dy=mat(4, 7)),
    "8-bit dy": dict(dy=f8(4, 8)),
    "8-bit dtable": dict(dtable=f8(9, 8)),
    "dtable over dy": dict(dy=mat(4, 8, ptr=8192), dtable=mat(4, 8, ptr=8192)),
    "no dtable": dict(dtable=mat(9, 8, ptr=0)),
    "misaligned dtable": dict(dtable=mat(9, 8, ptr=4098)),
    "dtable too short for its stride": dict(dtable=bf(9, 8, ld=64, nbytes=128)),
    "scale not finite": dict(scale=float("inf")),
    "an empty table": dict(dtable=mat(0, 8)),
}


@pytest.mark.parametrize("case", GRAD)
def test_embed_grad_refuses(vs, case):
    kw = dict(dy=mat(4, 8), ids=ids(4), dtable=mat(9, 8, ptr=65536))
    kw.update(GRAD[case])
    refused(vs, vs.VCSR_EINVAL, vs.run_embed_grad_gpu, **kw)


@pytest.mark.parametrize("ws", [f8(16), f8(1 << 24, ptr=4104)], ids=["short", "misaligned"])
@pytest.mark.parametrize("M", [65, 5000, 50000])
def test_embed_grad_refuses_a_workspace(vs, ws, M):
    refused(vs, vs.VCSR_EINVAL, vs.run_embed_grad_gpu, dy=mat(M, 8), ids=ids(M),
            dtable=mat(9, 8, ptr=1 << 30), workspace=ws)


def test_embed_null_arguments_and_sizes(vs):
    lib, need = vs.load_library(), C.c_size_t(0)
    for fn in ("vcsr_embed", "vcsr_embed_grad"):
        assert getattr(lib, fn)(None, None, None) == vs.VCSR_EINVAL, fn
    assert lib.vcsr_embed_grad_workspace(None, None) == vs.VCSR_EINVAL
    ok = dict(M=4, V=9, C=8, ids=4096, scale=1.0)
    for bad, code in ((dict(M=1 << 31), vs.VCSR_ERANGE), (dict(C=(1 << 20) + 1), vs.VCSR_ERANGE),
                      (dict(M=-1), vs.VCSR_EINVAL), (dict(V=0), vs.VCSR_EINVAL)):
        a = vs._EmbedArgs(table=4096, y=8192, **{**ok, **bad})
        assert lib.vcsr_embed(C.byref(a), None, None) == code, bad
        a = vs._EmbedGradArgs(dy=4096, dtable=8192, **{**ok, **bad})
        assert lib.vcsr_embed_grad(C.byref(a), None, None) == code, bad
        assert lib.vcsr_embed_grad_workspace(C.byref(a), C.byref(need)) == code, bad
    a = vs._EmbedGradArgs(dy=4096, dtable=8192, accumulate=2, **ok)
    assert lib.vcsr_embed_grad(C.byref(a), None, None) == vs.VCSR_EINVAL


def test_embed_without_a_gpu_says_so(vs):
    if vs.device_count() > 0:
        pytest.skip("a GPU is visible")
    refused(vs, vs.VCSR_EDEVICE, vs.run_embed_gpu, mat(9, 8), ids(4), mat(4, 8, ptr=65536))
    refused(vs, vs.VCSR_EDEVICE, vs.run_embed_grad_gpu, mat(4, 8), ids(4), bf(9, 8, ptr=65536))
