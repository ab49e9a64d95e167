"""The 8-bit cache's writer and its dense view, byte for byte against the restatement."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import hip_ops
from oracle import kv8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F8 = torch.float8_e4m3fn


def _pools(blocks, heads, dim, block, fill=0x2B):
    make = lambda: torch.full((blocks, heads, hip_ops.kv8_tile_bytes(dim, block)), fill, dtype=torch.uint8, device=DEV).view(F8)  # noqa: E731
    return make(), make()


def _bytes(pool):
    return pool.contiguous().view(torch.uint8).cpu().numpy().copy()


def _rows(gen, tokens, heads, dim, dtype):
    x = torch.randn(tokens, heads, dim, generator=gen) * torch.exp(3 * torch.randn(tokens, heads, 1, generator=gen))
    return x.to(dtype)


def _by_run(gen, slots, block):
    """Slots with the runs in random order, and the tokens of a run together, in random order."""
    runs = [slots[i : i + 16] for i in range(0, len(slots), 16)]
    out = []
    for i in torch.randperm(len(runs), generator=gen):
        run = runs[i]
        out.append(run[torch.randperm(len(run), generator=gen)])
    return torch.cat(out)


def _append_both(pools, host, key, value, slots, block):
    hip_ops.paged_kv8_append(key.to(DEV), value.to(DEV), *pools, slots.to(DEV), block)
    for pool, want, rows, is_key in zip(pools, host, (key, value), (True, False)):
        kv8.append(want, slots.numpy(), rows.double().numpy(), block, is_key)
        assert kv8.same_bytes(_bytes(pool), want, rows.shape[-1]), "keys" if is_key else "values"


@pytest.mark.parametrize("dim,block,heads", [(256, 16, 2), (128, 16, 1), (128, 64, 3), (256, 32, 1)])
@pytest.mark.parametrize("dtype,index", [(torch.bfloat16, torch.int64), (torch.float32, torch.int32)])
@pytest.mark.parametrize("tokens", [1, 16, 67, 1100])
def test_append_writes_the_bytes_of_the_format(dim, block, heads, dtype, index, tokens) -> None:
    gen = torch.Generator().manual_seed(dim + block + tokens)
    blocks = -(-tokens // block) + 2
    key, value = (_rows(gen, tokens, heads, dim, dtype) for _ in range(2))
    slots = _by_run(gen, torch.arange(blocks * block)[:tokens], block).to(index)
    if tokens > 20:
        # every 16th from 1 on lies outside the pool; its neighbours still belong together
        slots[5], slots[17], slots[21] = -1, blocks * block, -(1 << 30)
        key[0, 0, :3] = torch.tensor([0.0, -0.0, 1e-38]).to(dtype)
        key[4, 0, 32:64] = 0
        key[5, 0, 5], value[5, heads - 1, 70], value[6, 0, 3] = float("nan"), float("inf"), float("-inf")
        value[40, 0, :] = 3.0e38
        value[50:66, 0, :] = 1e-40
        key[50:66, 0, :] = float("nan")
        value[9, 0, :8] = torch.tensor([448.0, 450.0, -0.75, 1.25, -1.75, 2.5, 3.5, 5.0]).to(dtype)
    pools = _pools(blocks, heads, dim, block)
    _append_both(pools, [_bytes(p) for p in pools], key, value, slots, block)


@pytest.mark.parametrize("dim,block,heads,dtype", [(256, 16, 2, torch.bfloat16), (128, 64, 1, torch.float32), (128, 16, 2, torch.bfloat16)])
def test_runs_that_grow_call_by_call(dim, block, heads, dtype) -> None:
    """Tokens a few at a time, some of them far larger or far smaller than what their run holds, then the first ones again."""
    gen = torch.Generator().manual_seed(dim + block)
    pools = _pools(3, heads, dim, block, fill=0xFF)
    host = [_bytes(p) for p in pools]
    at = 0
    for step, count in enumerate((1, 1, 3, 1, 20, 1, 1, 2, 7, 1, 1, 1, 5)):
        count = min(count, 3 * block - at)
        if count <= 0:
            break
        key, value = (_rows(gen, count, heads, dim, dtype) * (1000.0 if step % 3 == 1 else 1e-6 if step % 4 == 2 else 1.0) for _ in range(2))
        if step == 5:
            key[:] = float("nan")
            value[:] = 0
        _append_both(pools, host, key.to(dtype), value.to(dtype), torch.arange(at, at + count), block)
        at += count
    for start, count in ((0, 1), (3, 2), (9, 7)):  # tokens taken back and written again
        _append_both(pools, host, *(_rows(gen, count, heads, dim, dtype) for _ in range(2)), torch.arange(start, start + count), block)


def test_a_batch_of_single_tokens_touches_their_runs_only() -> None:
    gen = torch.Generator().manual_seed(3)
    pools = _pools(40, 2, 256, 16)
    host = [_bytes(p) for p in pools]
    _append_both(pools, host, *(_rows(gen, 640, 2, 256, torch.bfloat16) for _ in range(2)), torch.arange(640), 16)
    for offset in (0, 7, 15):
        slots = torch.randperm(40, generator=gen)[:33] * 16 + offset
        slots[4] = -1
        _append_both(pools, host, *(_rows(gen, 33, 2, 256, torch.bfloat16) for _ in range(2)), slots, 16)


@pytest.mark.parametrize("gap", [130, 1100, 2300])
@pytest.mark.parametrize("front,tail", [(0, 0), (1, 70), (64, 5000), (1500, 1)])
def test_runs_with_long_stretches_of_skipped_tokens(gap, front, tail) -> None:
    """Padded slot maps: a run goes on behind the stretch, another begins there, and nothing follows the last."""
    gen = torch.Generator().manual_seed(gap + front)
    skipped = lambda n: torch.full((n,), -1, dtype=torch.int64)  # noqa: E731
    slots = torch.cat((skipped(front), torch.arange(3, 9), skipped(gap), torch.arange(9, 13), skipped(gap - 63), torch.tensor([13]), skipped(gap), torch.arange(32, 75), skipped(tail)))
    pools = _pools(6, 1, 128, 16)
    _append_both(pools, [_bytes(p) for p in pools], *(_rows(gen, slots.numel(), 1, 128, torch.bfloat16) for _ in range(2)), slots, 16)


def test_append_reads_strided_rows_in_place() -> None:
    gen = torch.Generator().manual_seed(5)
    both = torch.randn(20, 2, 512, generator=gen).to(torch.bfloat16).to(DEV)
    key, value = both[..., :256], both[:, :, 256:]
    slots = torch.arange(20, device=DEV)
    a, b = _pools(2, 2, 256, 16), _pools(2, 2, 256, 16)
    equal = lambda: all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))  # noqa: E731
    hip_ops.paged_kv8_append(key, value, *a, slots, 16)
    hip_ops.paged_kv8_append(key.contiguous(), value.contiguous(), *b, slots, 16)
    assert equal()
    odd = torch.randn(20, 2, 257, generator=gen).to(torch.bfloat16).to(DEV)[..., 1:]  # rows that cannot be read in 16-byte pieces
    hip_ops.paged_kv8_append(odd, odd, *a, slots, 16)
    hip_ops.paged_kv8_append(odd.contiguous(), odd.contiguous(), *b, slots, 16)
    assert equal()
    one = torch.randn(20, 1, 256, generator=gen).to(torch.bfloat16).to(DEV).expand(-1, 2, -1)  # a head for both
    hip_ops.paged_kv8_append(one, one, *a, slots, 16)
    hip_ops.paged_kv8_append(one.contiguous(), one.contiguous(), *b, slots, 16)
    assert equal()


@pytest.mark.parametrize("dim,block,heads,index", [(256, 16, 2, torch.int32), (128, 64, 3, torch.int64), (256, 32, 1, torch.int64)])
@pytest.mark.parametrize("valid", [1, 16, 77])
def test_gather_gives_the_values_the_cache_holds(dim, block, heads, index, valid) -> None:
    gen = torch.Generator().manual_seed(dim + valid)
    batch, need = 2, -(-valid // block)
    blocks = batch * need + 3
    pools = _pools(blocks, heads, dim, block, fill=0)
    tables = torch.randperm(blocks, generator=gen)[: batch * need].view(batch, need).to(index)
    tokens = torch.arange(valid)
    slots = tables.long()[:, tokens // block] * block + tokens % block
    key, value = (_rows(gen, batch * valid, heads, dim, torch.bfloat16) for _ in range(2))
    key[0, 0, 3] = float("nan")
    hip_ops.paged_kv8_append(key.to(DEV), value.to(DEV), *pools, slots.reshape(-1).to(DEV), block)
    held = [_bytes(p) for p in pools]
    if need > 1:
        tables[1, 1] = -1
        tables[0, need - 1] = blocks
    got = hip_ops.paged_kv8_gather(*pools, tables.to(DEV), valid, block)
    for out, pool, is_key in zip(got, held, (True, False)):
        want = np.zeros((batch, heads, valid, dim))
        for b in range(batch):
            for t in range(valid):
                if 0 <= int(tables[b, t // block]) < blocks:
                    for h in range(heads):
                        want[b, h, t] = kv8.read(pool, int(slots[b, t]), h, block, dim, is_key)
        assert out.dtype == torch.bfloat16 and tuple(out.shape) == want.shape
        assert np.array_equal(out.cpu().double().numpy(), want, equal_nan=True)


def test_gather_past_the_table_and_empty() -> None:
    kp, vp = _pools(2, 1, 128, 16, fill=0x7E)
    k, v = hip_ops.paged_kv8_gather(kp, vp, torch.tensor([[1]], device=DEV), 40, 16)
    assert not k[:, :, 16:].any() and not v[:, :, 16:].any()
    k, v = hip_ops.paged_kv8_gather(kp, vp, torch.tensor([1], device=DEV), 0, 16)
    assert k.shape == (1, 1, 0, 128)
    hip_ops.paged_kv8_append(torch.zeros(0, 1, 128, device=DEV), torch.zeros(0, 1, 128, device=DEV), kp, vp, torch.zeros(0, dtype=torch.int64, device=DEV), 16)


def test_pool_views_with_strides_of_their_own() -> None:
    tile = hip_ops.kv8_tile_bytes(256, 16)
    kp, vp = (torch.zeros(3, 4, tile + 16, dtype=torch.uint8, device=DEV).view(F8)[:, ::2, :tile] for _ in range(2))
    x = torch.randn(48, 2, 256, device=DEV).to(torch.bfloat16)
    slots = torch.arange(48, device=DEV)
    hip_ops.paged_kv8_append(x, -x, kp, vp, slots, 16)
    a, b = _pools(3, 2, 256, 16)
    hip_ops.paged_kv8_append(x, -x, a, b, slots, 16)
    table = torch.arange(3, device=DEV)
    for got, want in zip(hip_ops.paged_kv8_gather(kp, vp, table, 48, 16), hip_ops.paged_kv8_gather(a, b, table, 48, 16)):
        assert torch.equal(got, want)


def test_captured_append_replays_as_eager_runs() -> None:
    x = torch.randn(5, 2, 128, device=DEV).to(torch.bfloat16)
    slots = torch.tensor([3, 35, 16, 70, -1], device=DEV)
    a, b = _pools(6, 2, 128, 16, fill=0), _pools(6, 2, 128, 16, fill=0)
    hip_ops.paged_kv8_append(x, x, *a, slots, 16)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hip_ops.paged_kv8_append(x, x, *a, slots, 16)
    for p, q in zip(a, b):
        q.copy_(p)
    for step in range(5):
        x.mul_(-3.0)
        slots[slots >= 0] += 1
        hip_ops.paged_kv8_append(x, x, *b, slots, 16)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(a, b))


def test_refusals_of_tensors() -> None:
    kp, vp = _pools(2, 2, 256, 16)
    x = torch.zeros(3, 2, 256, dtype=torch.bfloat16, device=DEV)
    s = torch.zeros(3, dtype=torch.int64, device=DEV)
    for args in ((x, x, kp, vp, s, 32), (x[:, :1], x, kp, vp, s, 16), (x, x.float(), kp, vp, s, 16), (x.half(), x.half(), kp, vp, s, 16), (x, x, kp, vp, s[:2], 16),
                 (x, x, kp, vp, s.float(), 16), (x, x, kp.view(torch.uint8), vp, s, 16), (x, x, kp, vp[:1], s, 16), (x, x.cpu(), kp, vp, s, 16), (x[:2], x, kp, vp, s, 16)):
        with pytest.raises(RuntimeError):
            hip_ops.paged_kv8_append(*args)
