"""Which kernel a dense product takes, and calls that are made to take one (tests)."""
from __future__ import annotations

import contextlib
import ctypes as C

TYPE = {"f32": 0, "bf16": 1, "fp8": 2}
# (tile, stages) of each type's products by rows; gradients have no four stages.
TILES = {"f32": [(64, 2), (128, 2)], "bf16": [(64, 2), (64, 4), (128, 2), (256, 2)],
         "fp8": [(64, 2), (128, 2), (256, 2)]}
STEP = {"f32": 32, "bf16": 64, "fp8": 128}  # values of a step of the sum


@contextlib.contextmanager
def forced(vs, tile, stages=2, splits=1, rows=0, together=False):
    """This thread's products take the tile, the splits of the sum and the first `rows`
    rows by themselves (0: all), as far as they have them."""
    force = vs.load_library().vcsr_test_force_plan
    force.argtypes = [C.c_int32, C.c_int32, C.c_int32, C.c_int64, C.c_int32]
    force.restype = None
    caches = (vs._linear_bytes, vs._linear_grad_bytes)  # workspace sizes go by the plan
    force(tile, stages, splits, rows, 1 if together else 0)
    for cache in caches:
        cache.cache_clear()
    try:
        yield
    finally:
        force(0, 0, 0, 0, 0)
        for cache in caches:
            cache.cache_clear()


def linear_plan(vs, M, N, K, xk, yk="bf16", residual=False, z=False):
    """(tile, stages, splits, rows) of a forward product."""
    out = (C.c_int64 * 4)()
    a = vs._LinearArgs(M=M, N=N, K=K, x_type=TYPE[xk], y_type=TYPE[yk],
                       residual=16 if residual else None, z=16 if z else None)
    vs._check(vs.load_library().vcsr_test_linear_plan(C.byref(a), out))
    return tuple(out)


def grad_plan(vs, M, N, K, kind, act="gelu"):
    """(together, dw's tile, dw's splits, dx's tile, dx's splits)."""
    out = (C.c_int64 * 5)()
    a = vs._LinearGradArgs(M=M, N=N, K=K, x_type=TYPE[kind], y_type=TYPE[kind],
                           act=vs.ACTIVATIONS[act], z=16, dx=16, dw=16, dbias=16)
    vs._check(vs.load_library().vcsr_test_linear_grad_plan(C.byref(a), out))
    return tuple(out)
