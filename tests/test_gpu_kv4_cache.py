"""The 4-bit cache's writer and its dense view, byte for byte against the restatement."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import hip_ops
from oracle import kv4

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _pools(blocks, heads, dim, block, fill=0xAB):
    make = lambda: torch.full((blocks, heads, hip_ops.kv4_tile_bytes(dim, block)), fill, dtype=torch.uint8, device=DEV)  # noqa: E731
    return make(), make()


def _rows(gen, tokens, heads, dim, dtype):
    x = torch.randn(tokens, heads, dim, generator=gen) * torch.exp(3 * torch.randn(tokens, heads, 1, generator=gen))
    return x.to(dtype)


@pytest.mark.parametrize("dim,block,heads", [(256, 16, 2), (128, 16, 1), (128, 64, 3), (256, 32, 1)])
@pytest.mark.parametrize("dtype,index", [(torch.bfloat16, torch.int64), (torch.float32, torch.int32)])
@pytest.mark.parametrize("tokens", [1, 16, 67])
def test_append_writes_the_bytes_of_the_format(dim, block, heads, dtype, index, tokens) -> None:
    gen = torch.Generator().manual_seed(dim + block + tokens)
    blocks = -(-tokens // block) + 2
    key, value = (_rows(gen, tokens, heads, dim, dtype) for _ in range(2))
    slots = torch.randperm(blocks * block, generator=gen)[:tokens].to(index)
    if tokens > 3:
        slots[1], slots[2], slots[3] = -1, blocks * block, -(1 << 30)
        key[0, 0, :3] = torch.tensor([0.0, -0.0, 1e-38]).to(dtype)
        key[4, 0, 32:64] = 0  # a group of zeros
        key[5, 0, 5], value[5, heads - 1, 70], value[6, 0, 3] = float("nan"), float("inf"), float("-inf")
        value[7, 0, :32] = 3.0e38
        value[8, 0, :32] = 1e-40
        value[9, 0, :8] = torch.tensor([7.0, 0.25, -0.75, 1.25, -1.75, 2.5, 3.5, 5.0]).to(dtype)
        value[9, 0, 8:32] = 0
    kp, vp = _pools(blocks, heads, dim, block)
    hip_ops.paged_kv4_append(key.to(DEV), value.to(DEV), kp, vp, slots.to(DEV), block)
    for pool, rows, is_key in ((kp, key, True), (vp, value, False)):
        want = np.full(pool.shape, 0xAB, dtype=np.uint8)
        for n in range(tokens):
            for h in range(heads):
                kv4.write(want, int(slots[n]), h, block, rows[n, h].double().numpy(), is_key)
        got = pool.cpu().numpy()
        # -0 and what rounds to it: the sign of a zero code is free
        differ = got != want
        assert np.array_equal(got[differ] & 0x77, want[differ] & 0x77), "codes or scales differ"
        for half in (0, 4):
            g, w = got[differ] >> half & 15, want[differ] >> half & 15
            assert np.all((g == w) | ((g & 7) == 0) & ((w & 7) == 0))


def test_append_reads_strided_rows_in_place() -> None:
    gen = torch.Generator().manual_seed(5)
    both = torch.randn(20, 2, 512, generator=gen).to(torch.bfloat16).to(DEV)
    key, value = both[..., :256], both[:, :, 256:]
    slots = torch.arange(20, device=DEV)
    a, b = _pools(2, 2, 256, 16), _pools(2, 2, 256, 16)
    hip_ops.paged_kv4_append(key, value, *a, slots, 16)
    hip_ops.paged_kv4_append(key.contiguous(), value.contiguous(), *b, slots, 16)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    odd = torch.randn(20, 2, 257, generator=gen).to(torch.bfloat16).to(DEV)[..., 1:]  # rows that cannot be read in 16-byte pieces
    hip_ops.paged_kv4_append(odd, odd, *a, slots, 16)
    hip_ops.paged_kv4_append(odd.contiguous(), odd.contiguous(), *b, slots, 16)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dim,block,heads,index", [(256, 16, 2, torch.int32), (128, 64, 3, torch.int64), (256, 32, 1, torch.int64)])
@pytest.mark.parametrize("valid", [1, 16, 77])
def test_gather_gives_the_values_the_cache_holds(dim, block, heads, index, valid) -> None:
    gen = torch.Generator().manual_seed(dim + valid)
    batch, need = 2, -(-valid // block)
    blocks = batch * need + 3
    kp, vp = _pools(blocks, heads, dim, block, fill=0)
    tables = torch.randperm(blocks, generator=gen)[: batch * need].view(batch, need).to(index)
    tokens = torch.arange(valid)
    slots = tables.long()[:, tokens // block] * block + tokens % block
    key, value = (_rows(gen, batch * valid, heads, dim, torch.bfloat16) for _ in range(2))
    key[0, 0, 3] = float("nan")
    hip_ops.paged_kv4_append(key.to(DEV), value.to(DEV), kp, vp, slots.reshape(-1).to(DEV), block)
    if need > 1:
        tables[1, 1] = -1
        tables[0, need - 1] = blocks
    got = hip_ops.paged_kv4_gather(kp, vp, tables.to(DEV), valid, block)
    for out, rows in zip(got, (key, value)):
        want = torch.from_numpy(kv4.quantized(rows.double().numpy())).view(batch, valid, heads, dim).transpose(1, 2).clone()
        if need > 1:
            want[1, :, block : 2 * block] = 0
            want[0, :, (need - 1) * block :] = 0
        assert out.dtype == torch.bfloat16 and out.shape == want.shape
        assert np.array_equal(out.cpu().double().numpy(), want.numpy(), equal_nan=True)


def test_gather_past_the_table_and_empty() -> None:
    kp, vp = _pools(2, 1, 128, 16, fill=0x7F)
    k, v = hip_ops.paged_kv4_gather(kp, vp, torch.tensor([[1]], device=DEV), 40, 16)
    assert not k[:, :, 16:].any() and not v[:, :, 16:].any()
    k, v = hip_ops.paged_kv4_gather(kp, vp, torch.tensor([1], device=DEV), 0, 16)
    assert k.shape == (1, 1, 0, 128)
    hip_ops.paged_kv4_append(torch.zeros(0, 1, 128, device=DEV), torch.zeros(0, 1, 128, device=DEV), kp, vp, torch.zeros(0, dtype=torch.int64, device=DEV), 16)


def test_pool_views_with_strides_of_their_own() -> None:
    tile = hip_ops.kv4_tile_bytes(256, 16)
    kp = torch.zeros(3, 4, tile + 16, dtype=torch.uint8, device=DEV)[:, ::2, :tile]
    vp = torch.zeros(3, 4, tile + 16, dtype=torch.uint8, device=DEV)[:, ::2, :tile]
    x = torch.randn(48, 2, 256, device=DEV).to(torch.bfloat16)
    slots = torch.arange(48, device=DEV)
    hip_ops.paged_kv4_append(x, -x, kp, vp, slots, 16)
    a, b = _pools(3, 2, 256, 16)
    hip_ops.paged_kv4_append(x, -x, a, b, slots, 16)
    assert torch.equal(kp, a) and torch.equal(vp, b)


def test_refusals_of_tensors() -> None:
    kp, vp = _pools(2, 2, 256, 16)
    x = torch.zeros(3, 2, 256, dtype=torch.bfloat16, device=DEV)
    s = torch.zeros(3, dtype=torch.int64, device=DEV)
    for args in ((x, x, kp, vp, s, 32), (x[:, :1], x, kp, vp, s, 16), (x, x.float(), kp, vp, s, 16), (x.half(), x.half(), kp, vp, s, 16), (x, x, kp, vp, s[:2], 16),
                 (x, x, kp, vp, s.float(), 16), (x, x, kp.float(), vp, s, 16), (x, x, kp, vp[:1], s, 16), (x, x.cpu(), kp, vp, s, 16), (x[:2], x, kp, vp, s, 16)):
        with pytest.raises(RuntimeError):
            hip_ops.paged_kv4_append(*args)
