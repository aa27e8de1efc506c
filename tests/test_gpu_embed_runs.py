"""The embedding's gradient of up to 64 tokens, which each wave sorts by itself, on the GPU:
runs of equal ids of every length from the first token on, and around a wave's share."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_embed import GRAD, grad_once

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kinds", GRAD)
@pytest.mark.parametrize("first", [1, 2, 3, 7, 8, 9, 15, 16, 17, 33, 63, 64])
def test_embed_grad_of_runs_in_a_wave(gpu, kinds, first):
    """The lowest id, zero or not, `first` times; then runs that begin at, before and behind
    multiples of 8."""
    dk, tk = kinds.split()
    st, rng = gpu.Stream(), np.random.default_rng(first)
    for M in sorted({first, min(64, first + 9), 64}):
        for low, length in ((0, 1), (5, 1), (5, 7), (5, 8), (3, 9)):
            ids = np.concatenate([np.full(first, low), low + 1 + np.arange(64) // length])[:M]
            ids = rng.permutation(ids).astype(np.int32)
            print(f"embed grad runs {kinds} M={M} first={first} low={low} x{length}", flush=True)
            one = grad_once(gpu, st, np.random.default_rng(2), M, 75, 40, dk, tk, ids, length == 7)
            two = grad_once(gpu, st, np.random.default_rng(2), M, 75, 40, dk, tk, ids, length == 7)
            assert one.tobytes() == two.tobytes()


def test_embed_grad_of_padding_in_a_wave(gpu):
    """A run that padding follows, padding alone, and one token among it."""
    st = gpu.Stream()
    for ids in ([4] * 9 + [-1] * 55, [-1] * 64, [-1] * 30 + [0] + [9] * 33, [7] * 2 + [-1] * 6,
                [0] * 2, [6, 6]):
        ids = np.int32(ids)
        for tk, add in (("f32", False), ("bf16", True)):
            print(f"embed grad padding {ids[:3]} {tk}", flush=True)
            grad_once(gpu, st, np.random.default_rng(3), len(ids), 9, 300, "bf16", tk, ids, add)
