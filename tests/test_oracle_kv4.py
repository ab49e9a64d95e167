"""The 64-bit restatement of the 4-bit cache holds what its format promises."""

from __future__ import annotations

import numpy as np
import pytest

import hip_ops
from oracle import kv4


def test_every_code_reads_back_as_itself() -> None:
    for byte in (2, 100, 127, 252):
        for codes in ([0, 1, 2, 3, 4, 5, 6, 7], [8, 9, 10, 11, 12, 13, 14, 15]):
            x = kv4.dequantize_group(byte, codes * 4)
            got_byte, got = kv4.quantize_group(x)
            assert got_byte == byte
            assert np.array_equal(kv4.dequantize_group(got_byte, got), x)


def test_no_element_is_further_than_half_a_step_from_its_code() -> None:
    rng = np.random.default_rng(0)
    for scale in (1e-30, 1.0, 1e30):
        x = rng.standard_normal((50, 32)) * scale
        x[:, 0] = 7.0 * 2.0 ** rng.integers(-3, 3, 50) * scale  # the far end of what rounds to 6
        for row in x:
            byte, codes = kv4.quantize_group(row)
            step = 2.0 ** (byte - 127)
            a = np.abs(row) / step
            spacing = np.where(a < 2, 0.5, np.where(a < 4, 1.0, 2.0))
            assert np.all(np.abs(kv4.dequantize_group(byte, codes) - row) <= spacing / 2 * step * (1 + 1e-12))


def test_ties_go_to_the_even_code_and_limits_hold() -> None:
    x = np.zeros(32)
    x[:8] = (6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)
    byte, codes = kv4.quantize_group(x)
    assert byte == 127 and codes[:8] == [7, 0, 2, 2, 4, 4, 6, 6]
    assert kv4.quantize_group(np.zeros(32)) == (2, [0] * 32)
    assert kv4.quantize_group(np.full(32, 3.3e38))[0] == 252
    assert kv4.quantize_group(np.array([np.nan] + [1.0] * 31))[0] == 255
    assert np.isnan(kv4.dequantize_group(255, [0])).all()


def test_vectorised_form_is_the_scalar_one() -> None:
    rng = np.random.default_rng(1)
    x = rng.standard_normal((40, 32)) * np.exp(rng.standard_normal((40, 1)) * 20)
    x[3] = 0.0
    x[4, 5] = np.inf
    got = kv4.quantized(x)
    for row, want in zip(x, got):
        assert np.array_equal(kv4.dequantize_group(*kv4.quantize_group(row)), want, equal_nan=True)


@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("block", [16, 64])
def test_places_cover_a_tile_once(dim: int, block: int) -> None:
    for is_key in (True, False):
        places = []
        for t in range(block):
            for g in range(dim // 32):
                if is_key:
                    at, scale = kv4.key_place(dim, t, g)
                    places += list(range(at, at + 16)) + [scale]
                else:
                    codes, scale = kv4.value_places(dim, t, g)
                    places += codes + [scale]
        assert sorted(places) == list(range(kv4.tile_bytes(dim, block)))
    assert kv4.tile_bytes(dim, block) == hip_ops.kv4_tile_bytes(dim, block)


def test_write_and_read_are_inverse_on_representable_values() -> None:
    rng = np.random.default_rng(2)
    for dim in (128, 256):
        pool = np.zeros((3, 2, kv4.tile_bytes(dim, 32)), dtype=np.uint8)
        for is_key in (True, False):
            x = kv4.quantized(rng.standard_normal(dim))
            kv4.write(pool, 41, 1, 32, x, is_key)
            assert np.array_equal(kv4.read(pool, 41, 1, 32, dim, is_key), x)


@pytest.mark.parametrize("sections,interleaved", [((11, 11, 10), True), ((16, 24, 24), False), ((16, 8, 8), True), ((5,), True), ((0, 3, 2, 4), False), ((4, 0, 3), True)])
def test_axes_of_the_frequencies(sections: tuple[int, ...], interleaved: bool) -> None:
    axes = hip_ops.mrope_axes(sections, interleaved)
    assert axes == [kv4.mrope_axis(j, sections, interleaved) for j in range(sum(sections))]
    if not interleaved:
        assert [axes.count(a) for a in range(len(sections))] == list(sections)


def test_equal_positions_give_the_usual_rotation() -> None:
    rng = np.random.default_rng(3)
    x = rng.standard_normal((5, 2, 64))
    pos = np.array([0, 1, 7, 1000, 100000])
    one = kv4.norm_mrope(x, np.zeros(64), pos[None], (8,), False, 1e4, 1e-6)
    for sections, interleaved in (((3, 3, 2), True), ((2, 2, 4), False)):
        three = kv4.norm_mrope(x, np.zeros(64), np.stack([pos] * 3), sections, interleaved, 1e4, 1e-6)
        np.testing.assert_allclose(three, one, atol=1e-12)
    # turning by p and then by q is turning by p + q: the norm of an already normalised head changes nothing but eps
    assert np.allclose((one[..., :8] ** 2 + one[..., 8:16] ** 2), kv4.norm_mrope(x, np.zeros(64), 0 * pos[None], (8,), False, 1e4, 1e-6)[..., :8] ** 2 +
                       kv4.norm_mrope(x, np.zeros(64), 0 * pos[None], (8,), False, 1e4, 1e-6)[..., 8:16] ** 2)


def test_plan_in_parts_is_the_plan_in_one() -> None:
    free = [3, 5, 6, 8, 9, 11, 12, 13]
    code, tables, lengths, head, count, cu, starts, positions, slots = kv4.plan([[-1] * 4, [7, -1, -1, -1]], [0, 5], [9, 20], free, 0, 8, 16, 40, 8)
    assert (code, lengths, head, count, cu, starts) == (0, [9, 25], 2, 6, [0, 9, 29], [0, 5])
    assert tables == [[3, -1, -1, -1], [7, 5, -1, -1]]
    assert positions[9:29] == list(range(5, 25)) and slots[9] == 7 * 16 + 5 and slots[20] == 5 * 16
    assert positions[29:] == [-1] * 11
    step = kv4.plan([[-1] * 4, [7, -1, -1, -1]], [0, 5], [4, 0], free, 0, 8, 16, 40, 8)
    again = kv4.plan(step[1], step[2], [5, 20], free, step[3], step[4], 16, 40, 8)
    assert again[1] == tables and again[2] == lengths
    assert kv4.plan([[-1]], [0], [17], free, 0, 8, 16, 40, 8)[0] == 2
    assert kv4.plan([[-1] * 9], [0], [129], free, 0, 8, 16, 400, 8)[0] == 1
    assert kv4.plan([[-1] * 9], [0], [41], free, 0, 8, 16, 40, 8)[0] == 5
    assert kv4.plan([[-1] * 9], [-1], [4], free, 0, 8, 16, 40, 8)[0] == 4
    assert kv4.plan([[-1] * 9], [0], [4], free, 1, 8, 16, 40, 8)[0] == 3
