"""The restatement of the 8-bit cache, pinned by the format's landmarks and torch's own E4M3."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv8


def test_values_are_torchs_e4m3() -> None:
    want = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(kv8.VALUES, want, equal_nan=True)
    assert kv8.GRID[-1] == 448 and kv8.GRID[1] == 2.0**-9 and np.all(np.diff(kv8.GRID) > 0)


def test_codes_are_torchs_roundings() -> None:
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(20_000, generator=gen, dtype=torch.float32) * torch.exp(3 * torch.randn(20_000, generator=gen))
    ties = torch.from_numpy((kv8.GRID[1:] + kv8.GRID[:-1]) / 2).float()
    x = torch.cat((x.clamp(-448, 448), ties, -ties, torch.tensor([0.0, -0.0, 448.0, -448.0, 2.0**-10, 3 * 2.0**-10])))
    want = x.to(torch.float8_e4m3fn).double()
    assert np.array_equal(kv8.VALUES[kv8.encode(x.double().numpy(), 0)], want.numpy())
    assert list(kv8.encode(np.array([np.nan, np.inf, -np.inf]), 0)) == [127] * 3


@pytest.mark.parametrize("amax,e", [(448.0, 0), (np.nextafter(448.0, 1e9), 1), (0.0, -117), (1e-38, -117), (3.4e38, 120), (1.75, -8), (1.76, -7), (224.0, -1)])
def test_scale_exponents(amax, e) -> None:
    assert kv8.scale_exponent(amax) == e


@pytest.mark.parametrize("dim", [128, 256])
def test_layouts_hold_every_byte_once(dim) -> None:
    for is_key in (True, False):
        places = np.concatenate([kv8.code_places(dim, t, is_key) for t in range(16)])
        assert sorted(places) == list(range(16 * dim))


def test_a_growing_run_keeps_its_values() -> None:
    """A larger token moves the scale: the values before stay but for what becomes subnormal, off by half a step of 2^-9 of it."""
    rng = np.random.default_rng(1)
    for is_key in (True, False):
        pool = np.zeros((1, 1, kv8.tile_bytes(128, 16)), np.uint8)
        x = rng.standard_normal((3, 1, 128))
        kv8.append(pool, np.array([0, 1]), x[:2], 16, is_key)
        before = [kv8.read(pool, s, 0, 16, 128, is_key) for s in (0, 1)]
        assert all(np.all(np.abs(b - v) <= 2.0**-4 * np.abs(v) + 2.0**-18 * np.abs(x).max()) for b, v in zip(before, x[:2, 0]))
        kv8.append(pool, np.array([2]), 1000 * x[2:], 16, is_key)
        scale = 2.0 ** (int(pool[0, 0, 2048]) - 127)
        for s in (0, 1):
            assert np.all(np.abs(kv8.read(pool, s, 0, 16, 128, is_key) - before[s]) <= scale * 2.0**-10 + 0 * before[s])
        again = pool.copy()
        kv8.append(pool, np.array([0]), x[:1], 16, is_key)  # its first token written again: the run starts anew
        assert pool[0, 0, 2048] < again[0, 0, 2048]
