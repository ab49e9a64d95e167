"""A decode step that the pool or the tables have no room for: nothing is written, zeros come out, and check() raises."""

from __future__ import annotations

import pytest
import torch

import attention_runtime as ar
from decode_state import DeviceBatchPageTables, SharedKV4BlockPool, SharedKVBlockPool
from test_gpu_kv4_runtime import _config

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HEADS, KV_HEADS, DIM, BLOCK = 16, 2, 256, 16
MROPE = ar.RopeConfig(mrope_section=(11, 11, 10), mrope_interleaved=True)


def _bf(gen, *shape):
    return torch.randn(*shape, generator=gen).to(torch.bfloat16).to(DEV)


class _Batch:
    """Rows with 16 tokens (a full block) and 5, and one that holds no request, on a pool of three blocks."""

    def __init__(self, kind, seed=1):
        self.gen = torch.Generator().manual_seed(seed)
        make = SharedKV4BlockPool if kind == "4-bit" else SharedKVBlockPool
        self.pool = make(3, KV_HEADS, DIM, block_size=BLOCK, device=DEV)
        self.tables = DeviceBatchPageTables(self.pool, rows=3, max_blocks=4)
        self.config, self.runtime = _config(HEADS, KV_HEADS, DIM), ar.HotPathRuntime()
        self.weights = [_bf(self.gen, DIM) * 0.3 for _ in range(2)]
        rows = [self.tables.add_request(), self.tables.add_request()]
        step = self.tables.plan_prefill(rows, [16, 5])
        ar.full_attention_prefill_device(*self.projections(21), *self.weights, self.pool.key_blocks, self.pool.value_blocks, step, self.config, self.runtime, MROPE)

    def projections(self, n):
        return _bf(self.gen, n, HEADS * 2 * DIM), _bf(self.gen, n, KV_HEADS * DIM), _bf(self.gen, n, KV_HEADS * DIM)

    def layer(self, x, plan):
        return ar.full_attention_decode_step_device(*x, *self.weights, self.pool.key_blocks, self.pool.value_blocks, self.tables, self.config, self.runtime, MROPE, plan=plan)

    def state(self):
        t = self.tables
        return [x.clone() for x in (self.pool.key_blocks, self.pool.value_blocks, t.block_tables, t.sequence_lengths, t.allocator.free_state)]

    def exhaust(self):
        """All of the free blocks, so that the row at the end of its block cannot grow."""
        self.tables.allocator.free_state[1] = 0


@pytest.mark.parametrize("kind", ["4-bit", "bf16"])
def test_a_refused_step_writes_nothing_and_gives_zeros(kind) -> None:
    batch = _Batch(kind)
    free = batch.tables.allocator.free_state.clone()
    batch.exhaust()
    before = batch.state()
    out = batch.layer(batch.projections(3), batch.tables.plan_step())
    assert not out.any() and all(torch.equal(a, b) for a, b in zip(batch.state(), before))
    with pytest.raises(RuntimeError, match="exhausted"):
        batch.tables.check()
    batch.tables.allocator.free_state.copy_(free)
    out = batch.layer(batch.projections(3), batch.tables.plan_step())
    batch.tables.check()
    assert out[0].any() and out[1].any() and not out[2].any() and batch.tables.sequence_lengths.tolist() == [17, 6, 0]


def test_a_plan_of_the_allocator_serves_as_well() -> None:
    batch = _Batch("4-bit")
    x = batch.projections(3)
    t = batch.tables
    kept = batch.state()
    want = batch.layer(x, t.plan_step())
    for now, old in zip((batch.pool.key_blocks, batch.pool.value_blocks, t.block_tables, t.sequence_lengths, t.allocator.free_state), kept):
        now.copy_(old)
    plan = t.allocator.plan(t.block_tables, t.sequence_lengths, BLOCK, counts=t.step_counts, max_tokens=3, per_row=1)
    assert torch.equal(batch.layer(x, plan), want) and want[0].any()


def test_post_rotary_keys_of_a_refused_step() -> None:
    batch = _Batch("4-bit")
    batch.exhaust()
    before = batch.state()
    q, k, v = (_bf(batch.gen, 3, h, 1, DIM) for h in (HEADS, KV_HEADS, KV_HEADS))
    out = ar.full_attention_decode_device(q, None, k, v, batch.pool.key_blocks, batch.pool.value_blocks, batch.tables, batch.config, batch.runtime, plan=batch.tables.plan_step())
    assert not out.any() and all(torch.equal(a, b) for a, b in zip(batch.state(), before))


def test_a_graph_replayed_past_the_end_of_the_pool() -> None:
    """Row 0 takes the third block with its 17th token, row 1 asks for a fourth with its own 17th."""
    batch = _Batch("4-bit")
    x = batch.projections(3)
    kept = batch.state()
    warm = batch.layer(x, batch.tables.plan_step())
    assert warm[0].any()
    t = batch.tables
    for now, old in zip((batch.pool.key_blocks, batch.pool.value_blocks, t.block_tables, t.sequence_lengths, t.allocator.free_state), kept):
        now.copy_(old)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = batch.layer(x, t.plan_step())
    for step in range(14):
        before = batch.state()
        graph.replay()
        torch.cuda.synchronize()
        if step < 11:  # row 1: 5 + 11 tokens fill its block
            t.check()
            assert out[0].any() and out[1].any() and not out[2].any()
            continue
        assert not out.any() and all(torch.equal(a, b) for a, b in zip(batch.state(), before))
        with pytest.raises(RuntimeError, match="paged_kv_plan failed: shared KV pool exhausted"):
            t.check()
