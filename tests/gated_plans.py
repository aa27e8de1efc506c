"""Calls of the gated projection that are made to take a kernel, and which one a size
takes (tests)."""
from __future__ import annotations

import contextlib
import ctypes as C

import dense_plans
from dense_plans import TYPE


@contextlib.contextmanager
def forced(vs, *args, **kw):
    """dense_plans.forced for the gated projection's products, dx and dw."""
    caches = (vs._gated_bytes, vs._gated_grad_bytes)  # workspace sizes go by the plan
    with dense_plans.forced(vs, *args, **kw):
        for cache in caches:
            cache.cache_clear()
        try:
            yield
        finally:
            for cache in caches:
                cache.cache_clear()


def gated_plan(vs, M, N, K, xk, yk="bf16", z=False):
    """(tile, stages, splits, rows) of a forward product."""
    out = (C.c_int64 * 4)()
    a = vs._GatedArgs(M=M, N=N, K=K, x_type=TYPE[xk], y_type=TYPE[yk], z_gate=16 if z else None,
                      z_up=32 if z else None)
    vs._check(vs.load_library().vcsr_test_gated_plan(C.byref(a), out))
    return tuple(out)


def gated_grad_plan(vs, M, N, K, kind, dx=True, dw=True):
    """(together, dw's tile, dw's splits, dx's tile, dx's splits)."""
    out = (C.c_int64 * 5)()
    a = vs._GatedGradArgs(M=M, N=N, K=K, x_type=TYPE[kind], y_type=TYPE[kind],
                          dx=16 if dx else None, dw_gate=32 if dw else None,
                          dw_up=48 if dw else None)
    vs._check(vs.load_library().vcsr_test_gated_grad_plan(C.byref(a), out))
    return tuple(out)
