"""The step plan against the token-by-token restatement."""

from __future__ import annotations

import random

import pytest
import torch

import hip_ops
from oracle import kv4

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _case(seed, batch, new_hi, prefix_hi, block, extra_blocks=5, width_slack=2):
    rng = random.Random(seed)
    lengths = [rng.randint(0, prefix_hi) for _ in range(batch)]
    counts = [rng.choice((0, 1, rng.randint(0, new_hi))) for _ in range(batch)]
    have = [-(-n // block) for n in lengths]
    want = [-(-(n + c) // block) for n, c in zip(lengths, counts)]
    blocks = sum(want) + extra_blocks
    ids = rng.sample(range(blocks), blocks)
    width = max(want) + width_slack
    tables, at = [], 0
    for n in have:
        tables.append(ids[at : at + n] + [-1] * (width - n))
        at += n
    free = sorted(ids[at:])
    return lengths, counts, tables, [-7] * 3 + free, 3, len(free)


def _run(lengths, counts, tables, free, head, count, block, max_tokens, counts_dtype=torch.int32, scalar=None):
    dev = lambda x, dtype=torch.int32: torch.tensor(x, dtype=dtype, device=DEV)  # noqa: E731
    t, n, f, state, status = dev(tables), dev(lengths), dev(free), dev([head, count]), dev([99])
    plan = hip_ops.paged_kv_plan(t, n, dev(counts, counts_dtype) if scalar is None else scalar, f, state, status, block, max_tokens=max_tokens)
    return (int(status), t.tolist(), n.tolist(), *state.tolist(), plan.cu_seqlens.tolist(), plan.starts.tolist(), plan.positions.tolist(), plan.slots.tolist())


def _check(case, block, max_tokens, **kw):
    lengths, counts, tables, free, head, count = case
    want = kv4.plan(tables, lengths, counts, free, head, count, block, max_tokens, len(free))
    got = _run(lengths, counts, tables, free, head, count, block, max_tokens, **kw)
    for name, g, w in zip(("status", "tables", "lengths", "head", "count", "cu", "starts", "positions", "slots"), got, want):
        assert g == w, name
    return want[0]


@pytest.mark.parametrize("batch,new_hi,prefix_hi,block", [(1, 1, 0, 16), (1, 5000, 17, 16), (7, 40, 100, 16), (64, 100, 300, 32), (300, 3, 40, 64), (1025, 9, 20, 16), (5, 2, 1000, 1)])
@pytest.mark.parametrize("pad", [0, 23])
def test_plan_matches_the_restatement(batch, new_hi, prefix_hi, block, pad) -> None:
    case = _case(batch * 31 + block, batch, new_hi, prefix_hi, block)
    total = sum(case[1])
    assert _check(case, block, total + pad, counts_dtype=torch.int64 if pad else torch.int32) == 0


def test_plan_of_many_rows_and_many_tokens() -> None:
    assert _check(_case(1, 5000, 4, 20, 16), 16, 20001) == 0  # more rows than are looked up in LDS
    assert _check(_case(2, 61, 2000, 700, 16), 16, 61 * 2000) == 0


def test_one_count_for_every_row() -> None:
    lengths, counts, tables, free, head, count = _case(3, 9, 1, 50, 16, extra_blocks=12)
    counts = [1] * 9
    want = kv4.plan(tables, lengths, counts, free, head, count, 16, 9, len(free))
    assert _run(lengths, counts, tables, free, head, count, 16, 9, scalar=1)[1:] == want[1:]


@pytest.mark.parametrize("change,code", [("exhausted", 1), ("narrow", 2), ("corrupt", 3), ("negative", 4), ("overflow", 4), ("tokens", 5)])
def test_a_step_that_does_not_fit_takes_nothing(change, code) -> None:
    lengths, counts, tables, free, head, count = _case(4, 6, 60, 90, 16)
    counts = [c + 17 for c in counts]
    tables = [row + [-1, -1] for row in tables]
    free = free + list(range(1000, 1020))
    count += 20
    max_tokens = sum(counts) + 3
    if change == "exhausted":
        count = 2
    elif change == "narrow":
        tables = [row[:4] for row in tables]
        counts[2] = 80
        max_tokens += 80
    elif change == "corrupt":
        head = len(free)
    elif change == "negative":
        counts[1] = -1
    elif change == "overflow":
        lengths[1] = 2**31 - 5
    elif change == "tokens":
        max_tokens = sum(counts) - 1
    assert _check((lengths, counts, tables, free, head, count), 16, max_tokens) == code


def test_rows_with_holes_in_their_tables_get_no_slot() -> None:
    lengths, counts, tables, free, head, count = [20], [3], [[4, -1, -1]], [9], 0, 1
    assert _check((lengths, counts, tables, free, head, count), 16, 5) == 0


def test_no_tokens_at_all() -> None:
    assert _check(([0, 5], [0, 0], [[-1], [2]], [1], 0, 1), 16, 0) == 0


def test_captured_plan_replays_step_after_step() -> None:
    block, batch = 16, 5
    tables = torch.full((batch, 8), -1, dtype=torch.int32, device=DEV)
    lengths = torch.tensor([0, 3, 15, 16, 31], dtype=torch.int32, device=DEV)
    for row, n in enumerate([0, 1, 1, 1, 2]):
        tables[row, :n] = torch.arange(100 + 10 * row, 100 + 10 * row + n)
    free = torch.arange(60, dtype=torch.int32, device=DEV)
    state = torch.tensor([0, 60], dtype=torch.int32, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    counts = torch.tensor([1, 7, 1, 0, 2], dtype=torch.int32, device=DEV)
    want = (tables.tolist(), lengths.tolist(), 0, 60)
    before = [x.clone() for x in (tables, lengths, state)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        hip_ops.paged_kv_plan(tables, lengths, counts, free, state, status, block, max_tokens=16)
    torch.cuda.synchronize()
    for x, y in zip((tables, lengths, state), before):
        x.copy_(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan = hip_ops.paged_kv_plan(tables, lengths, counts, free, state, status, block, max_tokens=16)
    for _ in range(6):
        graph.replay()
        torch.cuda.synchronize()
        code, *want, cu, starts, positions, slots = kv4.plan(want[0], want[1], counts.tolist(), list(range(60)), want[2], want[3], block, 16, 60)
        assert int(status) == code == 0
        assert tables.tolist() == want[0] and lengths.tolist() == want[1] and state.tolist() == want[2:]
        assert [x.tolist() for x in plan] == [cu, starts, positions, slots]
        (torch.ones(64, device=DEV) * 2).sum().item()


@pytest.mark.parametrize("batch,per_row,block", [(1, 1, 16), (128, 1, 16), (9, 4, 16), (1030, 5, 32), (5000, 1, 16), (70, 100, 16)])
def test_entries_for_every_row(batch, per_row, block) -> None:
    """Rows without a new token keep their entries, at -1; the rest of the plan is the packed one's."""
    lengths, counts, tables, free, head, count = _case(batch + per_row, batch, per_row, 60, block)
    code, *want = kv4.plan(tables, lengths, counts, free, head, count, block, sum(counts), len(free))
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    t, n, state, status = dev(tables), dev(lengths), dev([head, count]), dev([99])
    plan = hip_ops.paged_kv_plan(t, n, dev(counts), dev(free), state, status, block, max_tokens=batch * per_row, per_row=per_row)
    assert int(status) == code == 0
    assert [t.tolist(), n.tolist(), *state.tolist(), plan.cu_seqlens.tolist(), plan.starts.tolist()] == want[:6]
    cu = want[4]
    for got, packed in ((plan.positions, want[6]), (plan.slots, want[7])):
        assert got.tolist() == [packed[cu[b] + x] if x < counts[b] else -1 for b in range(batch) for x in range(per_row)]


def test_a_row_with_more_tokens_than_entries_takes_nothing() -> None:
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    t, n, state, status = dev([[-1], [3]]), dev([0, 5]), dev([0, 2]), dev([0])
    plan = hip_ops.paged_kv_plan(t, n, dev([0, 3]), dev([1, 2]), state, status, 16, max_tokens=4, per_row=2)
    assert int(status) == 5 and n.tolist() == [0, 5] and state.tolist() == [0, 2] and plan.slots.tolist() == [-1] * 4 and plan.cu_seqlens.tolist() == [0, 0, 0]
    with pytest.raises(RuntimeError, match="batch"):
        hip_ops.paged_kv_plan(t, n, 1, dev([1, 2]), state, status, 16, max_tokens=4, per_row=3)
