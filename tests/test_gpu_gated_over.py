"""The gated projection's gradients written over what no product reads, on the GPU: dx and the
dw over dy and both z, dx alone over x, the dw alone over the weights; the bits of a call
whose buffers are apart."""
from __future__ import annotations

import numpy as np
import pytest

from block_ref import values
from dense_ref import Mat, vector

pytestmark = pytest.mark.gpu

# M x N, M x K and N x K of one size, so that each may lie over another; one row, several
# tiles, split sums.
SIZES = [1, 40, 129, 400]


@pytest.mark.parametrize("over", [dict(dx="dy"), dict(dx="z_gate"), dict(dx="z_up"),
                                  dict(dw_gate="dy"), dict(dw_up="z_gate"),
                                  dict(dx="dy", dw_gate="z_gate", dw_up="z_up"),
                                  dict(dx="x", dw=None), dict(dw_gate="w_gate", dw_up="w_up", dx=None),
                                  dict(dw_gate="w_up", dw_up="w_gate", dx=None)],
                         ids=lambda o: " ".join(f"{k}-{v}" for k, v in o.items()))
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n", SIZES)
def test_gated_grad_over_what_is_not_read(gpu, n, kind, over):
    vs, st = gpu, gpu.Stream()
    want_dx = over.get("dx", "apart") is not None
    want_dw = over.get("dw", "apart") is not None

    def call(over):
        rng = np.random.default_rng(n)
        m = {k: Mat(vs, st, values(rng, (n, n), kind, n ** -0.5 if k[0] == "w" else 1.0), kind)
             for k in ("dy", "x", "w_gate", "w_up", "z_gate", "z_up")}
        out = {k: m.get(over.get(k)) or Mat(vs, st, None, kind, shape=(n, n))
               for k in ("dx", "dw_gate", "dw_up")
               if (want_dx if k == "dx" else want_dw)}
        bias = {k: vector(vs, st, np.full(n, np.nan)) for k in ("dgate_bias", "dup_bias")}
        print(f"gated grad over {n} {kind} {over}", flush=True)
        vs.run_gated_grad_gpu(*(m[k].view for k in ("dy", "x", "w_gate", "w_up", "z_gate", "z_up")),
                              act="gelu", **{k: v.view for k, v in out.items()}, **bias, stream=st)
        st.sync()
        assert all(np.isfinite(v.values()).all() for v in out.values())
        return {k: v.codes().tobytes() for k, v in out.items()}, \
            {k: v.numpy(st).tobytes() for k, v in bias.items()}

    same = call(over) == call({})
    assert same
