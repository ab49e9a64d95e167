"""The 8-bit cache at the far end of its numbers: every finite value is held as a finite one."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import hip_ops
from oracle import kv8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dim,block", [(128, 16), (256, 32)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_largest_values_are_held_as_finite_ones(dim, block, dtype) -> None:
    """From 248 2^120 on the nearest code is 256, and 256 2^120 = 2^128 is no bfloat16: 240 it is."""
    gen = torch.Generator().manual_seed(dim)
    top = torch.finfo(dtype).max
    key, value = (torch.randn(40, 2, dim, generator=gen) for _ in range(2))
    for x in (key, value):
        x[3, 0, :6] = torch.tensor([top, -top, 248 * 2.0**120, -247 * 2.0**120, 240 * 2.0**120, 1e38])
        x[20, 1, 5] = -top                   # beside small values, and
        x[21, 1, 7], x[22, 1, 8] = float("nan"), float("inf")  # what is not finite stays a NaN
        x[38, 0] = top
    key, value = key.to(dtype), value.to(dtype)
    blocks = -(-40 // block)
    pools = [torch.zeros(blocks, 2, hip_ops.kv8_tile_bytes(dim, block), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2)]
    host = [p.view(torch.uint8).cpu().numpy().copy() for p in pools]
    at = 0
    for count in (3, 1, 36):  # a run that grows up to them, and whole ones
        part = slice(at, at + count)
        hip_ops.paged_kv8_append(key[part].to(DEV), value[part].to(DEV), *pools, torch.arange(at, at + count, device=DEV), block)
        for pool, want, rows, is_key in zip(pools, host, (key, value), (True, False)):
            kv8.append(want, np.arange(at, at + count), rows[part].double().numpy(), block, is_key)
            assert kv8.same_bytes(pool.view(torch.uint8).cpu().numpy(), want, dim)
        at += count
    for got, rows in zip(hip_ops.paged_kv8_gather(*pools, torch.arange(blocks, device=DEV), 40, block), (key, value)):
        held, given = got[0].transpose(0, 1).cpu().double(), rows.double()
        assert torch.equal(held.isfinite(), given.isfinite()) and not held.isinf().any()
        big = (given.abs() >= 248 * 2.0**120) & given.isfinite()
        assert torch.equal(held[big].abs(), torch.full_like(held[big], 240 * 2.0**120)) and big.sum() >= 4 + dim


def test_attention_over_the_largest_values_is_finite() -> None:
    """One token: its value, whatever its key's score is."""
    top = torch.finfo(torch.bfloat16).max
    pools = [torch.zeros(2, 1, hip_ops.kv8_tile_bytes(128, 16), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2)]
    x = torch.full((1, 1, 128), top, dtype=torch.bfloat16, device=DEV)
    hip_ops.paged_kv8_append(torch.ones_like(x), x, *pools, torch.zeros(1, dtype=torch.int64, device=DEV), 16)
    query = torch.ones(1, 2, 1, 128, dtype=torch.bfloat16, device=DEV)
    table, one = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    out = hip_ops.paged_attention_decode_kv8(query, table, *pools, one, 16)
    assert (out.double() == 240 * 2.0**120).all()
    cu = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    out = hip_ops.paged_attention_prefill_kv8(query[:, :, 0], cu, cu[:1], *pools, table, 16, max_new=1)
    assert (out.double() == 240 * 2.0**120).all()
