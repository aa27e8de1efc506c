"""Which sort the embedding's gradient takes, and that its digits cover all ids (CPU)."""
from __future__ import annotations

import pytest

from embed_plans import DIGITS, RANKS, WAVE, embed_grad_plan


@pytest.mark.parametrize("M, sort", [(1, WAVE), (64, WAVE), (65, RANKS), (12288, RANKS),
                                     (12289, DIGITS), (1 << 20, DIGITS), ((1 << 31) - 1, DIGITS)])
def test_sort_by_the_number_of_tokens(vs, M, sort):
    assert embed_grad_plan(vs, M, 1000, 64)[0] == sort


@pytest.mark.parametrize("V, digits", [(1, 1), (2, 1), (511, 1), (512, 2), ((1 << 18) - 1, 2),
                                       (1 << 18, 3), ((1 << 27) - 1, 3), (1 << 27, 4),
                                       ((1 << 31) - 1, 4)])
def test_digits_by_the_number_of_rows(vs, V, digits):
    """Keys are ids and V itself, of tokens outside the table."""
    sort, n, bits, tile, _ = embed_grad_plan(vs, 20000, V, 8)
    assert (sort, n) == (DIGITS, digits)
    assert 1 <= bits <= 9 and V < 1 << (n * bits)


@pytest.mark.parametrize("M", [12289, 65536, 65537, 131072, 131073, 524288, 524289, 1 << 30,
                               (1 << 31) - 1])
def test_tiles_of_a_digit(vs, M):
    """Four waves a tile, 64 keys a turn, and few counts to read."""
    tile = embed_grad_plan(vs, M, 1000, 64)[3]
    assert tile % 256 == 0 and (M + tile - 1) // tile <= (128 if tile < 2048 else 256)
    assert vs._embed_grad_bytes(M, 1000, 64, 0, 0, 0) > 2 * 4 * M
