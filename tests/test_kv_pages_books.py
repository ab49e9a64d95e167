"""What the calls on a batch's shared pages leave behind when they refuse, without a GPU."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from decode_state import DeviceBatchPageTables, LinearStatePool, SharedKV8BlockPool


class _Recorded:
    """An allocator that notes which of the books' calls were reached."""

    def __init__(self):
        self.calls = []

    def _note(self, call):
        self.calls.append(call)
        return SimpleNamespace(sources=torch.zeros(1, dtype=torch.int32), targets=torch.ones(1, dtype=torch.int32))

    def fork(self, *args):
        return self._note("fork")

    def compact(self, *args):
        return self._note("compact")

    def check(self, *args):
        pass


def test_pools_are_checked_before_the_books_change() -> None:
    """Host tensors are pools that no page can be copied in: neither call may get as far as the books."""
    pool = SharedKV8BlockPool(8, kv_heads=2, head_dim=128)
    tables = DeviceBatchPageTables(pool, rows=3, max_blocks=4)
    tables.add_request()
    tables.allocator = _Recorded()
    pools = [pool.key_blocks, pool.value_blocks]
    for call in (lambda: tables.fork_request(0, 1, pools), lambda: tables.compact(pools)):
        with pytest.raises(RuntimeError, match="must be CUDA"):
            call()
    assert tables.allocator.calls == [] and tables.active == [True, False, False]


def test_a_fork_of_states_that_cannot_be_copied_takes_no_slot() -> None:
    states = LinearStatePool(6, 1, 4, 4, 8, 4)
    slot = states.acquire()
    for _ in range(2):
        with pytest.raises(RuntimeError, match="must be CUDA"):
            states.fork(slot, 3)
        assert states.free_slots == [1, 2, 3, 4, 5]
    assert states.acquire() == 1
