"""How the embedding's gradient sorts a number of tokens (tests)."""
from __future__ import annotations

import ctypes as C

from dense_plans import TYPE

WAVE, RANKS, DIGITS = range(3)


def embed_grad_plan(vs, M, V, width, dk="bf16", tk="f32", accumulate=False):
    """(sort, digits, bits of a digit, keys of a tile, tokens of a chunk)."""
    out = (C.c_int64 * 5)()
    a = vs._EmbedGradArgs(M=M, V=V, C=width, table_type=TYPE[tk], y_type=TYPE[dk],
                          accumulate=1 if accumulate else 0)
    vs._check(vs.load_library().vcsr_test_embed_grad_plan(C.byref(a), out))
    return tuple(out)
