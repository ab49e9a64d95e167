"""Bookkeeping of 8-bit pools and of shared pages, and the dispatch ladder over 8-bit pools, without a GPU."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

import attention_runtime as ar
from decode_state import (
    DecodeState, DeviceBatchPageTables, DeviceBlockAllocator, FullAttentionCache, LinearStatePool, SharedKV4BlockPool, SharedKV8BlockPool, SharedKVBlockPool, is_kv4, kv4_head_dim, tile_bits,
    tile_head_dim,
)


def test_pool_geometry_and_free_list() -> None:
    pool = SharedKV8BlockPool(6, kv_heads=2, head_dim=128, block_size=32)
    assert tuple(pool.key_blocks.shape) == (6, 2, 32 * 129) and tile_bits(pool.key_blocks) == 8 and not is_kv4(pool.key_blocks) and pool.block_count == 6
    assert pool.allocate(2) == [0, 1]
    pool.release([0])
    assert pool.allocate(2) == [0, 2]
    assert tile_head_dim(pool.key_blocks, pool.value_blocks, 32) == 128 and tile_head_dim(pool.key_blocks, pool.value_blocks, 16) is None
    assert tile_head_dim(pool.key_blocks, pool.value_blocks, 24) is None and kv4_head_dim(pool.key_blocks, pool.value_blocks, 32) is None
    again = SharedKV8BlockPool.from_tensors(pool.key_blocks, pool.value_blocks, block_size=32, free_blocks=[5, 4])
    assert again.head_dim == 128 and again.free_blocks == [4, 5] and tile_bits(SharedKVBlockPool(1, 1, 4).key_blocks) == 0
    assert tile_head_dim(pool.key_blocks, SharedKV4BlockPool(6, 2, 128).key_blocks, 32) is None


@pytest.mark.parametrize("call", [
    lambda: SharedKV8BlockPool(0, 2, 128), lambda: SharedKV8BlockPool(2, 0, 128), lambda: SharedKV8BlockPool(2, 2, 64), lambda: SharedKV8BlockPool(2, 2, 128, block_size=24),
    lambda: SharedKV8BlockPool(2, 2, 128, block_size=8), lambda: SharedKV8BlockPool.from_tensors(*[SharedKV4BlockPool(2, 2, 128).key_blocks] * 2),
    lambda: SharedKV4BlockPool.from_tensors(*[SharedKV8BlockPool(2, 2, 128).key_blocks] * 2), lambda: SharedKV8BlockPool.from_tensors(torch.zeros(2, 2, 16, 128), torch.zeros(2, 2, 16, 128)),
])
def test_bad_pools_raise(call) -> None:
    with pytest.raises((ValueError, RuntimeError)):
        call()


def test_cpu_tensors_are_refused_and_leave_the_cache_as_it_was() -> None:
    cache = FullAttentionCache(block_size=16, shared_pool=SharedKV8BlockPool(4, 2, 128))
    x = torch.zeros(1, 2, 5, 128)
    with pytest.raises(RuntimeError, match="8-bit pool is written from GPU tensors"):
        cache.append_blocks(x, x)
    assert cache.valid == 0 and cache.block_table == [] and cache.append_calls == 0
    mapping = SimpleNamespace(layers=[SimpleNamespace(index=0, layer_type="full_attention")])
    state = DecodeState.empty(mapping, shared_pools={0: SharedKV8BlockPool(4, 2, 128)})
    assert state.kv_stats().estimated_total_bytes == 2 * 4 * 2 * 16 * 129


def test_releases_of_shared_blocks() -> None:
    allocator = DeviceBlockAllocator(6, device="cpu", free_blocks=[5])
    allocator.references[2] = 1
    assert allocator.release([3, 2, 0]) == [3, 0]
    assert allocator.free_blocks() == [0, 3, 5] and allocator.references.tolist() == [0] * 6
    assert allocator.release([2]) == [2] and allocator.release([]) == []
    for bad in ([2], [4, 4], [6], [-1]):
        with pytest.raises(ValueError, match="not already free"):
            allocator.release(bad)


def test_forks_releases_and_compactions_are_checked_on_the_host() -> None:
    pool = SharedKV8BlockPool(8, kv_heads=2, head_dim=128)
    tables = DeviceBatchPageTables(pool, rows=3, max_blocks=4)
    pools = [pool.key_blocks, pool.value_blocks]
    tables.add_request()
    for call, message in ((lambda: tables.fork_request(1, 1, pools), "holds no request"), (lambda: tables.fork_request(0, 0, pools), "positive"),
                          (lambda: tables.fork_request(-3, 1, pools), "holds no request"), (lambda: tables.fork_request(3, 1, pools), "holds no request"),
                          (lambda: tables.fork_request(0, 1, []), "8 blocks each"), (lambda: tables.fork_request(0, 1, pools[:1]), "own pool"),
                          (lambda: tables.fork_request(0, 1, [*pools, torch.zeros(7, 2)]), "8 blocks each"), (lambda: tables.compact(pools[1:]), "own pool"),
                          (lambda: tables.compact(pools, max_moves=-1), "non-negative"), (lambda: tables.release_requests([0, 0]), "distinct"),
                          (lambda: tables.release_requests([1]), "holds no request"), (lambda: tables.release_requests([3]), "holds no request")):
        with pytest.raises(ValueError, match=message):
            call()
    with pytest.raises(RuntimeError, match="3 rows needed, 2 hold"):
        tables.fork_request(0, 3, pools)
    assert tables.active == [True, False, False]
    tables.release_requests([])
    states = LinearStatePool(2, 1, 4, 4, 8, 4)
    with pytest.raises(RuntimeError, match="exhausted"):
        states.fork(0, 3)
    for slot, count, message in ((0, 0, "positive"), (0, 1, "holds no request"), (2, 1, "holds no request"), (-1, 1, "holds no request")):
        with pytest.raises(ValueError, match=message):
            states.fork(slot, count)
    assert states.free_slots == [0, 1]


class _Gpu:
    """What the ladder looks at, on no device."""

    def __init__(self, shape, dtype):
        self.shape, self.dtype, self.is_cuda = shape, dtype, True

    def dim(self):
        return len(self.shape)


@pytest.mark.parametrize("query,pool,dtype,reason", [
    ((1, 16, 1, 256), (9, 2, 4112), torch.bfloat16, "no_kernel"), ((1, 8, 1, 128), (9, 2, 2064), torch.bfloat16, "no_kernel"), ((1, 16, 1, 256), (9, 2, 4112), torch.float32, "shape"),
    ((1, 15, 1, 256), (9, 2, 4112), torch.bfloat16, "shape"), ((1, 34, 1, 256), (9, 2, 4112), torch.bfloat16, "shape"), ((1, 16, 1, 64), (9, 2, 1040), torch.bfloat16, "shape"),
    ((1, 16, 1, 256), (9, 2, 4096), torch.bfloat16, "shape"), ((1, 16, 1, 256), (9, 2, 16, 256), torch.bfloat16, "shape"),
])
def test_the_ladder_over_8_bit_pools(query, pool, dtype, reason) -> None:
    config = ar.parse_attention_config({"text_config": {
        "linear_num_key_heads": 1, "linear_num_value_heads": 1, "linear_key_head_dim": 4, "linear_value_head_dim": 4, "linear_conv_kernel_dim": 4, "num_attention_heads": 16,
        "num_key_value_heads": 2, "head_dim": 256, "attn_output_gate": True, "native_paged_attention": True}})
    blocks = _Gpu(pool, torch.float8_e4m3fn)
    assert ar.paged_attention_fallback_reason(config, _Gpu(query, dtype), blocks, blocks, seq_len=1, batched=False) == reason
    assert ar.paged_attention_fallback_reason(config, _Gpu(query, dtype), blocks, blocks, seq_len=2, batched=False) == "prefill_or_multitoken"
    assert ar.paged_attention_fallback_reason(config, _Gpu(query, dtype), blocks, blocks, seq_len=1, batched=True) == "per_request_pools"
    assert ar.paged_attention_fallback_reason(config, _Gpu(query, dtype), blocks, _Gpu(pool, torch.uint8), seq_len=1, batched=False) == "shape"
