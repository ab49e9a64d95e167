"""Pages forked, copied, freed and moved on the device, equal to the restatement with lists."""

from __future__ import annotations

import random

import pytest
import torch

import hip_ops
from oracle.pages import Books

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class Device:
    """Books on the device beside their restatement."""

    def __init__(self, seed, lengths, rows, width, capacity, block, scattered=True):
        rng = random.Random(seed)
        ids = list(range(capacity))
        if scattered:
            rng.shuffle(ids)
        tables = torch.full((rows, width), -1, dtype=torch.int32)
        held = []
        for row, n in enumerate(lengths):
            need = -(-n // block)
            held.append([ids.pop() for _ in range(need)])
            tables[row, :need] = torch.tensor(held[-1], dtype=torch.int32)
        free = sorted(ids)
        self.host = Books(block, capacity, held + [[] for _ in range(rows - len(lengths))], list(lengths) + [0] * (rows - len(lengths)), list(free))
        head = rng.randint(0, capacity - len(free))
        self.tables = tables.to(DEV)
        self.lengths = torch.tensor(self.host.lengths, dtype=torch.int32, device=DEV)
        self.free = torch.full((capacity,), -7, dtype=torch.int32, device=DEV)
        self.free[head : head + len(free)] = torch.tensor(free, dtype=torch.int32)
        self.state = torch.tensor([head, len(free)], dtype=torch.int32, device=DEV)
        self.references = torch.zeros(capacity, dtype=torch.int32, device=DEV)
        self.status = torch.full((1,), 99, dtype=torch.int32, device=DEV)

    def fork(self, pairs, dtype=torch.int32):
        rows = torch.tensor(pairs, dtype=dtype, device=DEV).view(-1, 2)
        return hip_ops.paged_kv_fork(self.tables, self.lengths, rows[:, 0], rows[:, 1], self.free, self.state, self.references, self.status, self.host.block)

    def release(self, rows, dtype=torch.int32):
        hip_ops.paged_kv_release(self.tables, self.lengths, torch.tensor(rows, dtype=dtype, device=DEV), self.free, self.state, self.references, self.status)

    def compact(self, max_moves):
        return hip_ops.paged_kv_compact(self.tables, self.free, self.state, self.references, self.status, max_moves=max_moves)

    def check(self, pages=None, want_pages=None, ordered=None):
        assert self.status.item() == 0
        for row, (ids, n) in enumerate(zip(self.host.rows, self.host.lengths)):
            assert self.tables[row].tolist() == ids + [-1] * (self.tables.shape[1] - len(ids)), row
            assert self.lengths[row].item() == n
        head, count = self.state.tolist()
        assert self.free[head : head + count].tolist() == self.host.free
        if ordered:
            assert head == 0 and (self.free[count:] == -1).all()
        want = torch.zeros(self.host.capacity, dtype=torch.int32)
        for block, n in self.host.references.items():
            want[block] = n
        assert torch.equal(self.references.cpu(), want)
        if pages is not None:
            got = list(zip(pages.sources.tolist(), pages.targets.tolist()))
            assert got == want_pages + [(-1, -1)] * (len(got) - len(want_pages))

    def snapshot(self):
        return [t.clone() for t in (self.tables, self.lengths, self.free, self.state, self.references)]


@pytest.mark.parametrize("block", [16, 64, 5])
@pytest.mark.parametrize("dtype,width", [(torch.int32, 70), (torch.int64, 70), (torch.int32, 4200)])
def test_forks_releases_and_compactions_in_any_order(block, dtype, width) -> None:
    """Small books, which one workgroup keeps, and tables too wide for that."""
    rng = random.Random(block)
    d = Device(block, [rng.randint(0, 300) for _ in range(12)], 40, width, 1200, block)
    for step in range(30):
        live = [r for r in range(40) if d.host.rows[r] or d.host.lengths[r]]
        empty = [r for r in range(40) if d.host.lengths[r] == 0 and not d.host.rows[r]]
        kind = rng.choice(("fork", "release", "compact"))
        if kind == "fork" and live and empty:
            targets = rng.sample(empty, min(len(empty), rng.randint(1, 9)))
            pairs = [(rng.choice(live + [-1]), t) for t in targets]
            if sum(d.host.lengths[s] % block > 0 for s, _ in pairs if s >= 0) > len(d.host.free):
                continue
            pages = d.fork(pairs, dtype)
            d.check(pages, d.host.fork(pairs))
        elif kind == "release" and live:
            rows = rng.sample(live, min(len(live), rng.randint(1, 5)))
            d.release(rows + [rows[0], -1, 400], dtype)  # one of them twice, two that are not there
            d.host.release(rows)
            d.check(ordered=True)
        elif kind == "compact":
            most = rng.choice((3, 600))
            pages = d.compact(most)
            d.check(pages, d.host.compact(most), ordered=True)
    d.release(list(range(40)))
    d.host.release(list(range(40)))
    d.check(ordered=True)
    assert len(d.host.free) == 1200 and not d.references.any()


def test_forks_of_full_rows_empty_rows_and_many_of_one() -> None:
    d = Device(1, [32, 0, 33, 15], 100, 4, 300, 16)
    pairs = [(0, 10), (1, 11), (3, 12), (-1, 13), (2, 14), (2, 15)] + [(2, 20 + i) for i in range(60)]
    d.check(d.fork(pairs), d.host.fork(pairs))
    pairs = [(30, 90), (12, 91)]  # a fork's fork
    d.check(d.fork(pairs), d.host.fork(pairs))
    assert d.fork([]).sources.shape == (0,)
    d.check()


@pytest.mark.parametrize("pairs,state,code", [
    ([(0, 4), (0, 5), (1, 6)], (0, 2), 1), ([(0, 1)], None, 6), ([(0, 4), (1, 4)], None, 6), ([(0, 8)], None, 6), ([(9, 4)], None, 6), ([(0, 4), (4, 5)], None, 6),
    ([(0, -1)], None, 6), ([(4, 4)], None, 6), ([(0, 4)], (5, 1 << 30), 3), ([(0, 4)], (-1, 3), 3),
])
def test_a_refused_fork_changes_nothing(pairs, state, code) -> None:
    d = Device(2, [20, 7, 33], 8, 4, 40, 16)
    if state:
        d.state.copy_(torch.tensor(state))
    before = d.snapshot()
    pages = d.fork(pairs)
    assert d.status.item() == code
    assert (pages.sources == -1).all() and (pages.targets == -1).all()
    assert all(torch.equal(a, b) for a, b in zip(before, d.snapshot()))


def test_a_length_that_the_table_does_not_hold_is_refused() -> None:
    for length in (65, -1):
        d = Device(3, [20], 4, 4, 40, 16)
        d.lengths[0] = length
        before = d.snapshot()
        d.fork([(0, 1)])
        assert d.status.item() == 4 and all(torch.equal(a, b) for a, b in zip(before, d.snapshot()))


def test_a_corrupt_cursor_refuses_releases_and_compactions() -> None:
    d = Device(4, [20, 7, 33], 8, 4, 40, 16)
    d.state.copy_(torch.tensor([39, 5]))
    before = d.snapshot()
    d.release([0, 1])
    assert d.status.item() == 3 and all(torch.equal(a, b) for a, b in zip(before, d.snapshot()))
    d.status.zero_()
    pages = d.compact(10)
    assert d.status.item() == 3 and all(torch.equal(a, b) for a, b in zip(before, d.snapshot())) and (pages.sources == -1).all()


def test_compaction_leaves_blocks_of_others_where_they_are() -> None:
    d = Device(5, [100, 200, 50], 3, 20, 200, 16)
    others = d.host.free[-20:]  # taken by a holder that these tables do not know
    d.host.free = d.host.free[:-20]
    d.state[1] -= 20
    pages = d.compact(100)
    d.check(pages, d.host.compact(100), ordered=True)
    assert not set(others) & set(d.host.free) and not set(others) & set(pages.sources.tolist())
    again = d.compact(100)
    assert (again.sources == -1).all()
    d.check(ordered=True)
    assert d.compact(0).sources.shape == (0,)


@pytest.mark.parametrize("capacity", [1, 31, 32, 33, 2047, 8193, 32_768, 32_769, 34_817, 100_003])
def test_lists_of_any_length(capacity) -> None:
    """Words and workgroups that the list's end does not fill."""
    n = min(capacity, 70)
    d = Device(capacity, [1] * n, n + 2, 2, capacity, 16)
    pages = d.compact(capacity)
    d.check(pages, d.host.compact(capacity), ordered=True)
    d.release([0, n - 1, n])
    d.host.release([0] + ([n - 1] if n > 1 else []))
    d.check(ordered=True)


def test_copies_of_pages_of_every_kind() -> None:
    gen = torch.Generator(device=DEV).manual_seed(6)
    pools = [torch.randn(50, 2, 16, 256, generator=gen, device=DEV).to(torch.bfloat16), torch.randint(0, 255, (50, 2, 4112), generator=gen, device=DEV, dtype=torch.uint8),
             torch.randint(0, 255, (60, 1, 2176), generator=gen, device=DEV, dtype=torch.uint8), torch.randn(50, 4, 128, 128, generator=gen, device=DEV),
             torch.randn(50, 9000, generator=gen, device=DEV)]
    pools[1] = pools[1].view(torch.float8_e4m3fn)
    bits = lambda p: p.view(torch.uint8) if p.element_size() == 1 else p  # noqa: E731
    for index in (torch.int32, torch.int64):
        ids = torch.randperm(50, generator=gen, device=DEV)
        sources, targets = ids[:20].to(index), ids[25:45].to(index)
        sources[3], targets[5], sources[7], targets[8] = -1, -1, 60, 1 << 30
        sources[9] = sources[10]  # one page to two places
        want = []
        for p in pools:
            w = bits(p).clone()
            ok = [(int(s), int(t)) for s, t in zip(sources, targets) if 0 <= s < p.shape[0] and 0 <= t < p.shape[0]]
            for s, t in ok:
                w[t] = bits(p)[s]
            want.append(w)
        hip_ops.paged_kv_copy(pools, sources, targets)
        assert all(torch.equal(bits(p), w) for p, w in zip(pools, want))
    # pages that lie apart, and units of 4 bytes
    wide = torch.zeros(8, 40, device=DEV)
    part = wide[:, 4:33]
    part.copy_(torch.randn(8, 29, generator=gen, device=DEV))
    kept = wide.clone()
    hip_ops.paged_kv_copy([part], torch.tensor([1], device=DEV), torch.tensor([6], device=DEV))
    kept[6, 4:33] = kept[1, 4:33]
    assert torch.equal(wide, kept)
    many = [torch.randn(4, 8, generator=gen, device=DEV) for _ in range(70)]  # more than a launch takes
    want = [torch.stack((m[0], m[1], m[2], m[0])) for m in many]
    hip_ops.paged_kv_copy(many, torch.tensor([0], device=DEV), torch.tensor([3], device=DEV))
    assert all(torch.equal(m, w) for m, w in zip(many, want))
    hip_ops.paged_kv_copy(many, torch.zeros(0, dtype=torch.int32, device=DEV), torch.zeros(0, dtype=torch.int32, device=DEV))


def test_copies_of_pages_of_more_pieces_than_a_launch_has_workgroups() -> None:
    """Pages of 80 MB and of 64 bytes in one call, and so many small ones that a workgroup takes several."""
    gen = torch.Generator(device=DEV).manual_seed(8)
    for big in (20_000_003 // 4 * 4, 20_000_001):  # units of 16 and of 4 bytes
        pools = [torch.randn(3, big, generator=gen, device=DEV), torch.randn(3, 16, generator=gen, device=DEV)]
        want = [torch.stack((p[0], p[0], p[2])) for p in pools]
        hip_ops.paged_kv_copy(pools, torch.tensor([0, 7], device=DEV), torch.tensor([1, 2], device=DEV))
        assert all(torch.equal(p, w) for p, w in zip(pools, want))
    pools = [torch.randn(20_000, 2, 9, generator=gen, device=DEV), torch.randn(20_000, 5000, generator=gen, device=DEV).to(torch.bfloat16)]
    ids = torch.randperm(20_000, generator=gen, device=DEV)
    sources, targets = ids[:9000], ids[10_000:19_000]
    want = [p.clone() for p in pools]
    for w in want:
        w[targets] = w[sources]
    hip_ops.paged_kv_copy(pools, sources, targets)
    assert all(torch.equal(p, w) for p, w in zip(pools, want))


def test_copies_past_four_gigabytes() -> None:
    pool = torch.empty(5 * 2**30 // 8192, 4096, dtype=torch.bfloat16, device=DEV)
    pool[0] = 1.5
    last = pool.shape[0] - 1
    pool[last] = 0
    hip_ops.paged_kv_copy([pool], torch.tensor([0, last - 1], device=DEV), torch.tensor([last, 5], device=DEV))
    assert (pool[last] == 1.5).all()


def test_captured_fork_copy_and_release_replay_as_eager_runs() -> None:
    """Parallel sampling in a graph: children forked, their last pages copied, the children freed again."""
    block, rows = 16, 8
    pools = [torch.randn(64, 2, block, 128, device=DEV).to(torch.bfloat16) for _ in range(2)]
    d = Device(7, [40, 100], rows, 8, 64, block)
    source, target = torch.tensor([0, 0, 1], device=DEV), torch.tensor([3, 4, 5], device=DEV)

    def step(d, pools):
        pages = hip_ops.paged_kv_fork(d.tables, d.lengths, source, target, d.free, d.state, d.references, d.status, block)
        hip_ops.paged_kv_copy(pools, pages.sources, pages.targets)
        forked = d.tables.clone()
        hip_ops.paged_kv_release(d.tables, d.lengths, target, d.free, d.state, d.references, d.status)
        moved = hip_ops.paged_kv_compact(d.tables, d.free, d.state, d.references, d.status, max_moves=16)
        hip_ops.paged_kv_copy(pools, moved.sources, moved.targets)
        return forked, pages, moved

    step(d, pools)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        forked, pages, moved = step(d, pools)
    for turn in range(5):
        other = Device(7, [40, 100], rows, 8, 64, block)
        for a, b in zip((other.tables, other.lengths, other.free, other.state, other.references), (d.tables, d.lengths, d.free, d.state, d.references)):
            if turn % 2:
                b.copy_(a)  # the scattered start again
            else:
                a.copy_(b)
        copies = [p.clone() for p in pools]
        want = step(other, copies)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(forked, want[0]) and d.status.item() == 0
        for got, ref in ((pages, want[1]), (moved, want[2])):
            assert torch.equal(got.sources, ref.sources) and torch.equal(got.targets, ref.targets)
        assert all(torch.equal(a, b) for a, b in zip(d.snapshot(), other.snapshot()))
        assert all(torch.equal(a, b) for a, b in zip(pools, copies))


def test_refusals_of_tensors() -> None:
    d = Device(8, [20], 4, 4, 40, 16)
    rows = torch.zeros(1, dtype=torch.int32, device=DEV)
    fork = lambda **k: hip_ops.paged_kv_fork(*[k.get(n, v) for n, v in dict(t=d.tables, l=d.lengths, s=rows, r=rows + 1, f=d.free, c=d.state, h=d.references, u=d.status).items()], 16)  # noqa: E731
    for bad in (dict(t=d.tables.long()), dict(t=d.tables[0]), dict(l=d.lengths[:3]), dict(s=rows.float()), dict(s=rows.repeat(2)), dict(r=rows.long()), dict(f=d.free.long()), dict(c=d.state[:1]),
                dict(h=d.references[:5]), dict(u=d.status.long()), dict(s=rows.cpu(), r=rows.cpu()), dict(s=rows.repeat(1025), r=rows.repeat(1025))):
        with pytest.raises(RuntimeError):
            fork(**bad)
    with pytest.raises(RuntimeError):
        d.compact(-1)
    pool = torch.zeros(4, 8, device=DEV)
    for bad in (([], rows, rows), ([pool[:, ::2]], rows, rows), ([pool.cpu()], rows, rows), ([pool], rows.float(), rows.float()), ([pool], rows, rows.long()), ([pool[0]], rows, rows),
                ([torch.zeros(4, 3, dtype=torch.bfloat16, device=DEV)], rows, rows), ([pool[:1].expand(4, -1)], rows, rows)):
        with pytest.raises(RuntimeError):
            hip_ops.paged_kv_copy(*bad)
