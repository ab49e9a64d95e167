"""What the calls on a batch's shared pages leave behind when they refuse, without a GPU."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

import hip_ops
from decode_state import DeviceBatchPageTables, DeviceBlockAllocator, LinearStatePool, SharedKV8BlockPool


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


def _answers(monkeypatch, **codes):
    """Each operator on the books writes its status, as the kernels do: the code given for it, or 0."""
    def operator(name, status_at, gives):
        def call(*args, **kwargs):
            args[status_at].fill_(codes.get(name, 0))
            return gives
        monkeypatch.setattr(hip_ops, name, call)

    copies = hip_ops.PagedCopy(torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    for name, status_at, gives in (("paged_kv_reserve", 4, None), ("paged_kv_plan", 5, None), ("paged_kv_fork", 7, copies), ("paged_kv_release", 6, None), ("paged_kv_compact", 4, copies)):
        operator(name, status_at, gives)
    return codes


PAGE_CALLS = {
    "paged_kv_fork": lambda a: a.fork(None, None, None, None, 16),
    "paged_kv_release": lambda a: a.release_rows(None, None, None),
    "paged_kv_compact": lambda a: a.compact(None, 1),
}


@pytest.mark.parametrize("step", ["paged_kv_plan", "paged_kv_reserve"])
def test_a_refused_step_is_told_whatever_runs_behind_it(monkeypatch, step) -> None:
    codes = _answers(monkeypatch, **{step: 1})
    allocator = DeviceBlockAllocator(6, device="cpu")
    run = (lambda: allocator.plan(None, None, 16, max_tokens=1)) if step == "paged_kv_plan" else (lambda: allocator.reserve(None, None, 16))
    run()
    for call in PAGE_CALLS.values():
        call(allocator)
    for _ in range(2):  # until the next step
        with pytest.raises(RuntimeError, match=f"{step} failed: shared KV pool exhausted"):
            allocator.check()
    codes[step] = 0
    run()
    allocator.check()


@pytest.mark.parametrize("name", PAGE_CALLS)
def test_a_refused_page_call_is_told_whatever_runs_behind_it(monkeypatch, name) -> None:
    codes = _answers(monkeypatch, **{name: 3})
    allocator = DeviceBlockAllocator(6, device="cpu")
    PAGE_CALLS[name](allocator)
    codes[name] = 0
    for other in PAGE_CALLS:
        if other != name:
            PAGE_CALLS[other](allocator)
    allocator.plan(None, None, 16, max_tokens=1)
    with pytest.raises(RuntimeError, match=f"{name} failed: device free list state is corrupt"):
        allocator.check()
    allocator.check()  # once


def test_a_reservation_that_is_checked_at_once_answers_for_itself(monkeypatch) -> None:
    """A page call's refusal that nobody has looked at yet is no failure of an admission, nor the other way round."""
    codes = _answers(monkeypatch, paged_kv_fork=1)
    pool = SharedKV8BlockPool(8, kv_heads=2, head_dim=128)
    tables = DeviceBatchPageTables(pool, rows=3, max_blocks=4)
    PAGE_CALLS["paged_kv_fork"](tables.allocator)
    assert tables.add_request(prompt_tokens=5) == 0
    tables.reserve_prefill([0], [3])
    with pytest.raises(RuntimeError, match="paged_kv_fork failed"):
        tables.check()
    codes.update(paged_kv_fork=0, paged_kv_reserve=1)
    tables.reserve_step()
    monkeypatch.setattr(hip_ops, "page_pools", lambda pools: pools)
    monkeypatch.setattr(hip_ops, "paged_kv_copy", lambda *args: None)
    assert tables.fork_request(0, 1, [pool.key_blocks, pool.value_blocks]) == [1]
    with pytest.raises(RuntimeError, match="paged_kv_reserve failed"):
        tables.check()
    codes["paged_kv_fork"] = 1
    with pytest.raises(RuntimeError, match="paged_kv_fork failed"):
        tables.fork_request(0, 1, [pool.key_blocks, pool.value_blocks])
    codes["paged_kv_reserve"] = 0
    tables.reserve_step()
    tables.check()  # the fork has been told
    assert tables.active == [True, True, False]


def test_releases_on_the_host_behind_a_cursor() -> None:
    """The list's front has been taken, and blocks have up to three holders."""
    allocator = DeviceBlockAllocator(9, device="cpu")
    allocator.free_state.copy_(torch.tensor([5, 4]))  # 0 to 4 are held
    allocator.references[:5] = torch.tensor([0, 2, 1, 0, 0], dtype=torch.int32)
    assert allocator.release([4, 1, 2]) == [4]
    assert allocator.free_blocks() == [4, 5, 6, 7, 8] and allocator.references.tolist() == [0, 1, 0] + [0] * 6
    assert allocator.release([2, 1, 0]) == [2, 0]
    assert allocator.release([1]) == [1]
    assert allocator.free_blocks() == [0, 1, 2, 4, 5, 6, 7, 8] and not allocator.references.any() and allocator.free_state.tolist() == [0, 8]
    with pytest.raises(ValueError, match="not already free"):
        allocator.release([3, 8])
