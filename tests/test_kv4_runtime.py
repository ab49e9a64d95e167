"""Bookkeeping of 4-bit pools and the dispatch ladder over them, without a GPU."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

import attention_runtime as ar
from decode_state import DeviceBatchPageTables, DecodeState, FullAttentionCache, SharedKV4BlockPool, SharedKVBlockPool, is_kv4, kv4_head_dim


def test_pool_geometry_and_free_list() -> None:
    pool = SharedKV4BlockPool(6, kv_heads=2, head_dim=128, block_size=32)
    assert tuple(pool.key_blocks.shape) == (6, 2, 32 * 17 * 4) and is_kv4(pool.key_blocks) and pool.block_count == 6
    assert pool.allocate(2) == [0, 1]
    pool.release([0])
    assert pool.allocate(2) == [0, 2]
    with pytest.raises(RuntimeError, match="exhausted"):
        pool.allocate(4)
    assert kv4_head_dim(pool.key_blocks, pool.value_blocks, 32) == 128 and kv4_head_dim(pool.key_blocks, pool.value_blocks, 16) == 256
    assert kv4_head_dim(pool.key_blocks, pool.value_blocks, 64) is None and kv4_head_dim(pool.key_blocks, pool.value_blocks, 24) is None
    again = SharedKV4BlockPool.from_tensors(pool.key_blocks, pool.value_blocks, block_size=32, free_blocks=[5, 4])
    assert again.head_dim == 128 and again.free_blocks == [4, 5] and not is_kv4(SharedKVBlockPool(1, 1, 4).key_blocks)


@pytest.mark.parametrize("call", [
    lambda: SharedKV4BlockPool(0, 2, 128), lambda: SharedKV4BlockPool(2, 0, 128), lambda: SharedKV4BlockPool(2, 2, 64), lambda: SharedKV4BlockPool(2, 2, 128, block_size=24),
    lambda: SharedKV4BlockPool(2, 2, 128, block_size=8), lambda: SharedKV4BlockPool.from_tensors(torch.zeros(2, 2, 100, dtype=torch.uint8), torch.zeros(2, 2, 100, dtype=torch.uint8)),
    lambda: SharedKV4BlockPool.from_tensors(torch.zeros(2, 2, 16, 128), torch.zeros(2, 2, 16, 128)),
])
def test_bad_pools_raise(call) -> None:
    with pytest.raises((ValueError, RuntimeError)):
        call()


def test_cpu_tensors_are_refused_and_leave_the_cache_as_it_was() -> None:
    cache = FullAttentionCache(block_size=16, shared_pool=SharedKV4BlockPool(4, 2, 128))
    x = torch.zeros(1, 2, 5, 128)
    with pytest.raises(RuntimeError, match="GPU tensors"):
        cache.append_blocks(x, x)
    assert cache.valid == 0 and cache.block_table == [] and cache.append_calls == 0
    with pytest.raises(ValueError, match="block size"):
        FullAttentionCache(block_size=32, shared_pool=SharedKV4BlockPool(4, 2, 128))
    mapping = SimpleNamespace(layers=[SimpleNamespace(index=0, layer_type="full_attention")])
    state = DecodeState.empty(mapping, shared_pools={0: SharedKV4BlockPool(4, 2, 128)})
    assert state.kv_stats().estimated_total_bytes == 2 * 4 * 2 * 16 * 17 * 4


def test_step_rows_of_a_plan() -> None:
    pool = SharedKV4BlockPool(8, kv_heads=2, head_dim=128)
    tables = DeviceBatchPageTables(pool, rows=3, max_blocks=4)
    assert [tables.add_request(), tables.add_request()] == [0, 1]
    for rows, counts, message in (([], [], "one count per row"), ([0], [1, 2], "one count per row"), ([0, 0], [1, 1], "distinct"), ([3], [1], "distinct"), ([0], [0], "positive"),
                                  ([2], [1], "holds no request"), ([1, 0], [1, 1], "ascending")):
        with pytest.raises(ValueError, match=message):
            tables.plan_prefill(rows, counts)
    with pytest.raises(RuntimeError):  # the operators take GPU tensors
        tables.plan_prefill([0, 1], [3, 4])


class _Gpu:
    """What the ladder looks at, on no device."""

    def __init__(self, shape, dtype):
        self.shape, self.dtype, self.is_cuda = shape, dtype, True

    def dim(self):
        return len(self.shape)


@pytest.mark.parametrize("query,pool,dtype,reason", [
    ((1, 16, 1, 256), (9, 2, 2176), torch.bfloat16, "no_kernel"), ((1, 8, 1, 128), (9, 2, 1088), torch.bfloat16, "no_kernel"), ((1, 16, 1, 256), (9, 2, 2176), torch.float32, "shape"),
    ((1, 15, 1, 256), (9, 2, 2176), torch.bfloat16, "shape"), ((1, 34, 1, 256), (9, 2, 2176), torch.bfloat16, "shape"), ((1, 16, 1, 64), (9, 2, 544), torch.bfloat16, "shape"),
    ((1, 16, 1, 256), (9, 2, 2000), torch.bfloat16, "shape"), ((1, 16, 1, 256), (9, 2, 16, 256), torch.bfloat16, "shape"),
])
def test_the_ladder_over_4_bit_pools(query, pool, dtype, reason) -> None:
    config = ar.parse_attention_config({"text_config": {
        "linear_num_key_heads": 1, "linear_num_value_heads": 1, "linear_key_head_dim": 4, "linear_value_head_dim": 4, "linear_conv_kernel_dim": 4, "num_attention_heads": 16,
        "num_key_value_heads": 2, "head_dim": 256, "attn_output_gate": True, "native_paged_attention": True}})
    blocks = _Gpu(pool, torch.uint8)
    assert ar.paged_attention_fallback_reason(config, _Gpu(query, dtype), blocks, blocks, seq_len=1, batched=False) == reason
    assert ar.paged_attention_fallback_reason(config, _Gpu(query, dtype), blocks, blocks, seq_len=2, batched=False) == "prefill_or_multitoken"
    assert ar.paged_attention_fallback_reason(config, _Gpu(query, dtype), blocks, blocks, seq_len=1, batched=True) == "per_request_pools"


def test_rotary_sections() -> None:
    assert ar.RopeConfig().sections(256) == (32,) and ar.RopeConfig(mrope_section=(11, 11, 10)).sections(256) == (11, 11, 10)
