"""The dense operators on the GPU where lifetimes, limits and shared buffers matter."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from conftest import capture, hip_runtime
from dense_ref import Mat, pack

pytestmark = pytest.mark.gpu


def test_a_graph_outlives_the_workspace_it_was_captured_with(gpu):
    """A product whose sum is split, captured with the binding's workspace; then an eager
    call that needs a larger one, and buffers of the outgrown one's size: replays
    write none of them and give the eager call's bits."""
    vs, st = gpu, gpu.Stream()
    hip = hip_runtime()
    rng = np.random.default_rng(70)
    lib = vs.load_library()
    vs.release_workspaces()

    def product(M, N, K):
        x, w = rng.standard_normal((M, K)), rng.standard_normal((N, K)) / np.sqrt(K)
        X, W = Mat(vs, st, x, "f32"), Mat(vs, st, w, "f32")
        return X, W, Mat(vs, st, None, "f32", shape=(M, N)), x

    X, W, Y, x = product(64, 64, 8000)
    assert vs._linear_bytes(64, 64, 8000, 0, 0, False, False) > 0

    def step():
        vs.run_linear_gpu(X.view, W.view, Y.view, stream=st)

    step()
    st.sync()
    small = vs.workspace(1, st)
    graph, kinds = capture(hip, st, step)
    gexec = ctypes.c_void_p()
    try:
        assert kinds and all(k == 0 for k in kinds), kinds
        assert hip.hipGraphInstantiateWithFlags(ctypes.byref(gexec), graph, 0) == 0
        # A wide gradient: dz alone is larger than the first workspace.
        M, N, K = 3000, 512, 64
        dy, z, xx = (Mat(vs, st, rng.standard_normal((M, n)), "f32") for n in (N, N, K))
        ww, dx = Mat(vs, st, rng.standard_normal((N, K)), "f32"), \
            Mat(vs, st, None, "f32", shape=(M, K))
        vs.run_linear_grad_gpu(dy.view, xx.view, ww.view, z=z.view, act="silu", dx=dx.view,
                               stream=st)
        st.sync()
        large = vs.workspace(1, st)
        assert large is not small and large.nbytes > small.nbytes
        guards = [vs.DeviceArray.from_numpy(np.full(small.nbytes, 0x5B, np.uint8), st)
                  for _ in range(3)]
        for n in range(3):
            values = x * (n + 1)
            host = X.host.copy()
            X.grid(host)[:, :X.cols] = pack(values, "f32")
            vs._check(lib.vcsr_memcpy_h2d(X.buf.ptr, host.ctypes.data, host.nbytes, st.h))
            step()
            st.sync()
            eager = Y.codes().tobytes()
            Y.buf.copy_from(vs.DeviceArray.from_numpy(Y.host, st), st)
            st.sync()
            print(f"replay {n}", flush=True)
            assert hip.hipGraphLaunch(gexec, st.h) == 0
            st.sync()
            assert Y.codes().tobytes() == eager
            assert all((g.numpy(st) == 0x5B).all() for g in guards)
    finally:
        if gexec.value:
            hip.hipGraphExecDestroy(gexec)
        hip.hipGraphDestroy(graph)
    vs.release_workspaces()
