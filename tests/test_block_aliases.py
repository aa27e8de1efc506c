"""Embedding, layer norm, gated projection: outputs over vectors that the call reads, or
over each other, are refused before any device work (CPU)."""
from __future__ import annotations

import numpy as np
import pytest

from test_dense_refusals import Fake, bf, f8, mat, refused

P = [1 << 20 << i for i in range(20)]


def ids(n, **kw):
    return Fake((n,), np.int32, **kw)


def over(vs, fn, pairs, kw):
    """Each pair's second argument takes the buffer of its first."""
    for a, b in pairs:
        at = dict(kw)
        other = at[b]
        at[b] = Fake(other.shape, other.dtype, ptr=at[a].ptr.value)
        with pytest.raises(vs.VcsrError) as e:
            fn(**at)
        assert e.value.code == vs.VCSR_EINVAL, (a, b, e.value)


def apart(vs, fn, kw):
    """The same call with buffers of its own passes the checks: what is missing is a device."""
    if vs.device_count() == 0:
        refused(vs, vs.VCSR_EDEVICE, fn, **kw)


def test_embed(vs):
    kw = dict(table=f8(9, 8, ptr=P[0]), table_scale=mat(9, ptr=P[1]), ids=ids(4, ptr=P[2]),
              y=mat(4, 8, ptr=P[3]))
    over(vs, vs.run_embed_gpu, [("ids", "y"), ("table_scale", "y"), ("table", "y")], kw)
    apart(vs, vs.run_embed_gpu, kw)


@pytest.mark.parametrize("M", [40, 5000])
def test_embed_grad(vs, M):
    kw = dict(dy=mat(M, 8, ptr=P[0]), ids=ids(M, ptr=P[1]), dtable=mat(9, 8, ptr=P[2]),
              workspace=f8(1 << 24, ptr=P[10]))
    pairs = [("ids", "dtable"), ("dy", "dtable")]
    if M > 64:
        pairs += [(k, "workspace") for k in ("dy", "ids", "dtable")]
    over(vs, vs.run_embed_grad_gpu, pairs, kw)
    apart(vs, vs.run_embed_grad_gpu, kw)


VECTORS = ("weight", "bias")


def test_layernorm(vs):
    kw = dict(x=mat(8, 8, ptr=P[0]), residual=mat(8, 8, ptr=P[1]), weight=mat(8, ptr=P[2]),
              bias=mat(8, ptr=P[3]), sum=mat(8, 8, ptr=P[4]), y=f8(8, 8, ptr=P[5]),
              y_scale=mat(8, ptr=P[6]), mean=mat(8, ptr=P[7]), rstd=mat(8, ptr=P[8]))
    pairs = [(v, m) for v in VECTORS for m in ("sum", "y", "y_scale", "mean", "rstd")]
    pairs += [("mean", "rstd"), ("mean", "y_scale"), ("rstd", "y_scale")]
    pairs += [(m, v) for m in ("x", "residual", "sum", "y") for v in ("mean", "rstd", "y_scale")]
    over(vs, vs.run_layernorm_gpu, pairs, kw)
    apart(vs, vs.run_layernorm_gpu, kw)


@pytest.mark.parametrize("M, C", [(8, 8), (1, 20000), (5000, 8)])
def test_layernorm_grad(vs, M, C):
    kw = dict(dy=mat(M, C, ptr=P[0]), s=mat(M, C, ptr=P[1]), weight=mat(C, ptr=P[2]),
              mean=mat(M, ptr=P[3]), rstd=mat(M, ptr=P[4]), dsum=mat(M, C, ptr=P[5]),
              dx=mat(M, C, ptr=P[6]), dweight=mat(C, ptr=P[7]), dbias=mat(C, ptr=P[8]),
              workspace=f8(1 << 24, ptr=P[10]))
    read = ("weight", "mean", "rstd")
    pairs = [(v, "dx") for v in read] + [("dweight", "dbias")]
    pairs += [(v, d) for v in (*read, "dy", "s", "dsum", "dx") for d in ("dweight", "dbias")]
    if vs._layernorm_grad_bytes(M, C, 0, 0, True, True):
        pairs += [(k, "workspace") for k in kw if k != "workspace"]
    over(vs, vs.run_layernorm_grad_gpu, pairs, kw)
    apart(vs, vs.run_layernorm_grad_gpu, kw)


def test_gated(vs):
    kw = dict(x=f8(64, 8, ptr=P[0]), w_gate=f8(64, 8, ptr=P[1]), w_up=f8(64, 8, ptr=P[2]),
              y=mat(64, 64, ptr=P[3]), z_gate=mat(64, 64, ptr=P[4]), z_up=mat(64, 64, ptr=P[5]),
              x_scale=mat(64, ptr=P[6]), gate_scale=mat(64, ptr=P[7]), up_scale=mat(64, ptr=P[8]),
              gate_bias=mat(64, ptr=P[9]), up_bias=mat(64, ptr=P[10]),
              workspace=f8(1 << 26, ptr=P[15]))
    pairs = [(v, m) for v in ("x_scale", "gate_scale", "up_scale", "gate_bias", "up_bias")
             for m in ("y", "z_gate", "z_up")]
    over(vs, vs.run_gated_gpu, pairs, kw)
    apart(vs, vs.run_gated_gpu, kw)


def test_gated_over_its_workspace(vs):
    """A sum that is split."""
    M, N, K = 64, 64, 100000
    kw = dict(x=bf(M, K, ptr=P[0]), w_gate=bf(N, K, ptr=P[5]), w_up=bf(N, K, ptr=P[6]),
              y=bf(M, N, ptr=P[7]), z_gate=bf(M, N, ptr=P[8]), z_up=bf(M, N, ptr=P[9]),
              gate_bias=mat(N, ptr=P[10]), up_bias=mat(N, ptr=P[11]),
              workspace=f8(1 << 28, ptr=P[15]))
    assert vs._gated_bytes(M, N, K, 1, 1, True) > 0
    over(vs, vs.run_gated_gpu, [(k, "workspace") for k in kw if k != "workspace"], kw)
    apart(vs, vs.run_gated_gpu, kw)


@pytest.mark.parametrize("products", [True, False])
@pytest.mark.parametrize("M", [8, 5000])
def test_gated_grad(vs, M, products):
    N = K = 8
    kw = dict(dy=mat(M, N, ptr=P[0]), x=mat(M, K, ptr=P[1]), w_gate=mat(N, K, ptr=P[2]),
              w_up=mat(N, K, ptr=P[3]), z_gate=mat(M, N, ptr=P[4]), z_up=mat(M, N, ptr=P[5]),
              dgate_bias=mat(N, ptr=P[9]), dup_bias=mat(N, ptr=P[10]),
              workspace=f8(1 << 26, ptr=P[15]))
    if products:
        kw.update(dx=mat(M, K, ptr=P[6]), dw_gate=mat(N, K, ptr=P[7]), dw_up=mat(N, K, ptr=P[8]))
    mats = [k for k in ("dy", "z_gate", "z_up", "dx", "dw_gate", "dw_up") if k in kw]
    read = (["x", "w_gate", "w_up"] if products else [])
    pairs = [(m, b) for m in mats + read for b in ("dgate_bias", "dup_bias")]
    pairs.append(("dgate_bias", "dup_bias"))
    need = vs._gated_grad_bytes(M, N, K, 0, 0, products, products, True, True)
    if need:
        pairs += [(k, "workspace") for k in mats + read + ["dgate_bias", "dup_bias"]]
    over(vs, vs.run_gated_grad_gpu, pairs, kw)
    apart(vs, vs.run_gated_grad_gpu, kw)


def test_what_may_lie_over_inputs_still_does(vs):
    """dz is formed before the gated products: dx and the dw over dy or a z; layer norm's sum
    and y over x or the residual; no rows."""
    if vs.device_count() > 0:
        pytest.skip("a GPU is visible")
    kw = dict(dy=mat(8, 8, ptr=P[0]), x=mat(8, 8, ptr=P[1]), w_gate=mat(8, 8, ptr=P[2]),
              w_up=mat(8, 8, ptr=P[3]), z_gate=mat(8, 8, ptr=P[4]), z_up=mat(8, 8, ptr=P[5]),
              workspace=f8(1 << 26, ptr=P[15]))
    for k in ("dy", "z_gate", "z_up"):
        refused(vs, vs.VCSR_EDEVICE, vs.run_gated_grad_gpu, dx=kw[k], **kw)
    for s, y in (("x", "residual"), ("residual", "x")):
        kw = dict(x=mat(8, 8, ptr=P[0]), residual=mat(8, 8, ptr=P[1]), weight=mat(8, ptr=P[2]))
        refused(vs, vs.VCSR_EDEVICE, vs.run_layernorm_gpu, sum=kw[s], y=kw[y], **kw)
    none = mat(0, 8, ptr=0)
    refused(vs, vs.VCSR_EDEVICE, vs.run_layernorm_grad_gpu, none, none, mat(8, ptr=P[0]),
            mat(0, ptr=0), mat(0, ptr=0), none, mat(8, ptr=P[1]), mat(8, ptr=P[2]))
