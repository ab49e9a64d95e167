"""The books of a running batch around its page calls: what a refused call leaves, and what a later one may not hide."""

from __future__ import annotations

import pytest
import torch

from decode_state import DeviceBatchPageTables, SharedKVBlockPool

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _batch(blocks=12, rows=4, tokens=(40, 20)):
    pool = SharedKVBlockPool(blocks, 2, 128, device=DEV)
    tables = DeviceBatchPageTables(pool, rows=rows, max_blocks=6)
    for n in tokens:
        tables.add_request(prompt_tokens=n)
    return pool, tables


def _books(tables):
    a = tables.allocator
    return [t.clone() for t in (tables.block_tables, tables.sequence_lengths, tables.step_counts, a.free_list, a.free_state, a.references)]


BAD = {
    "host memory": lambda n: torch.zeros(n, 8),
    "one axis": lambda n: torch.zeros(n, device=DEV),
    "pages that are not contiguous": lambda n: torch.zeros(n, 16, device=DEV)[:, ::2],
    "pages of 6 bytes": lambda n: torch.zeros(n, 3, dtype=torch.bfloat16, device=DEV),
    "pages 10 bytes apart": lambda n: torch.zeros(n, 5, dtype=torch.bfloat16, device=DEV)[:, :4],
    "an odd address": lambda n: torch.zeros(8 * n + 1, dtype=torch.bfloat16, device=DEV)[1:].view(n, 8),
    "pages on top of each other": lambda n: torch.zeros(1, 8, device=DEV).expand(n, -1),
    "pages of nothing": lambda n: torch.zeros(n, 0, device=DEV),
}


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("alike", [False, True])
def test_pools_that_cannot_be_copied_leave_the_books_alone(bad, alike) -> None:
    """With a bad pool beside the batch's own, and beside one of its own kind."""
    pool, tables = _batch()
    tables.release_request(0)  # blocks 0 to 2 are free, so that a compaction has something to move
    pools = [pool.key_blocks, pool.value_blocks] + [BAD[bad](pool.block_count) for _ in range(1 + alike)]
    before, active = _books(tables), list(tables.active)
    with pytest.raises(RuntimeError):
        tables.compact(pools)
    with pytest.raises(RuntimeError):
        tables.fork_request(1, 2, pools)
    assert tables.active == active and all(torch.equal(a, b) for a, b in zip(before, _books(tables)))
    tables.compact(pools[:2])
    assert tables.block_tables[1, :2].tolist() == [1, 0] and tables.fork_request(1, 1, pools[:2]) == [0]


def test_a_refused_step_is_told_behind_releases_forks_and_compactions() -> None:
    pool, tables = _batch(blocks=5, tokens=(32, 32))  # a step of both needs two blocks, and there is one
    pools = [pool.key_blocks, pool.value_blocks]
    tables.plan_step()
    assert tables.fork_request(0, 1, pools) == [2]  # of full blocks alone
    tables.compact(pools)
    tables.release_requests([0, 2])
    for _ in range(2):
        with pytest.raises(RuntimeError, match="paged_kv_plan failed: shared KV pool exhausted"):
            tables.check()
    assert tables.sequence_lengths.tolist() == [0, 32, 0, 0]
    plan = tables.plan_step()
    tables.check()
    assert tables.sequence_lengths.tolist() == [0, 33, 0, 0] and plan.slots.tolist()[1] >= 0


def test_a_refused_fork_is_told_behind_a_step() -> None:
    pool, tables = _batch(blocks=5, tokens=(40, 20))  # no block is left for a partly filled last one
    a = tables.allocator
    rows = torch.tensor([0, 2], dtype=torch.int32, device=DEV)
    a.fork(tables.block_tables, tables.sequence_lengths, rows[:1], rows[1:], tables.block_size)
    tables.release_requests([])
    tables.plan_step()
    with pytest.raises(RuntimeError, match="paged_kv_fork failed: shared KV pool exhausted"):
        tables.check()
    tables.check()
    assert tables.sequence_lengths.tolist() == [41, 21, 0, 0]
