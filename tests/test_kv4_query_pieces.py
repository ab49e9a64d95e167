"""The query as two E4M3 pieces: what their sum and the fixed-point sums of eight products keep."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv4

MANTISSAS = np.arange(128, 256) / 128.0


def _rows(top_mantissa: float, below: int) -> np.ndarray:
    """Groups of eight dims with one element of the top's power of two and seven ``below`` binades under it, all mantissas."""
    small = np.concatenate([MANTISSAS, -MANTISSAS]) * 2.0**-below
    small = np.concatenate([small, np.zeros(-len(small) % 7)]).reshape(-1, 7)
    return np.concatenate([np.full((len(small), 1), top_mantissa), small], axis=1).reshape(-1)


@pytest.mark.parametrize("top", [1.0, 129 / 128, 1.9375, 255 / 128])
def test_the_pieces_are_e4m3_and_their_sum_is_the_element(top) -> None:
    for below in range(0, 30):
        row = _rows(top, below)
        if np.abs(row).max() != top:  # the small ones are larger than the top
            continue
        hi, lo, scale = kv4.query_pieces(row)
        for piece in (hi, lo):
            assert np.array_equal(torch.from_numpy(piece).to(torch.float8_e4m3fn).double().numpy(), piece)
        off = np.abs(scale * (hi + lo / 16) - row)
        exact = np.abs(row) >= 2.0**-7 * top
        assert not off[exact].any() and (off <= 2.0**-15 * top).all()


def test_groups_far_below_the_rows_largest_element() -> None:
    for below in range(5, 40):
        row = np.concatenate([[1.0] + [0.0] * 7, _rows(1.0, 3) * 2.0**-below])
        hi, lo, scale = kv4.query_pieces(row)
        off = np.abs(scale * (hi + lo / 16) - row)
        assert (off <= max(2.0**-15 * 2.0**-below, 2.0**-21)).all()


@pytest.mark.parametrize("top", [1.0, 1.5, 1.9375, 255 / 128])
def test_no_product_of_the_first_piece_has_places_below_the_cut(top) -> None:
    """Products of a group are cut 13 binades under the largest sum of their factors' exponents: at the least, that of
    a code of 4 or 6 at its largest element; codes are multiples of a half."""
    rng = np.random.default_rng(0)
    for _ in range(200):
        row = np.exp(rng.uniform(-12, 0, 64)) * rng.choice((-1, 1), 64)
        row = torch.from_numpy(row).to(torch.bfloat16).double().numpy()
        row[::8] = top
        hi, _, _ = kv4.query_pieces(row)
        for group in hi.reshape(-1, 8):
            unit = 2.0 ** (np.floor(np.log2(np.abs(group).max())) + 2 - 13)
            assert np.array_equal(np.rint(group * 0.5 / unit) * unit, group * 0.5)
