"""The 4-bit attention where rows are long enough to be split: that every token counts once, and everything that the short
rows are tested for where partial results are written and merged."""

from __future__ import annotations

import pytest
import torch

import hip_ops
from test_gpu_attention_kv4 import _attend, _cache, _close, _dense

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _together(total):
    """Tokens that share a mark: one in a row of up to 5000, else a run of 16."""
    return 1 if total <= 5000 else 16


def _marks(total, dim, gen):
    """The dim of each token, each dim about as often."""
    kinds = -(-total // _together(total))
    return (torch.randperm(kinds, generator=gen) % dim)[torch.arange(total) // _together(total)]


def _marked(totals, kv_heads, dim, block, seed):
    """A pool whose keys are 0 and whose token t of a row has a 1 at dim ``mark[t]`` of its values and zeros elsewhere."""
    gen = torch.Generator().manual_seed(seed)
    need = [-(-n // block) for n in totals]
    order = torch.randperm(sum(need), generator=gen).to(torch.int32)
    tables = torch.full((len(totals), max(need)), -1, dtype=torch.int32)
    at = 0
    for row, n in enumerate(need):
        tables[row, :n] = order[at : at + n]
        at += n
    pools = [torch.zeros(sum(need), kv_heads, hip_ops.kv4_tile_bytes(dim, block), dtype=torch.uint8, device=DEV) for _ in range(2)]
    marks = [_marks(n, dim, gen) for n in totals]
    for row, (n, mark) in enumerate(zip(totals, marks)):
        t = torch.arange(n)
        slots = (tables[row].long()[t // block] * block + t % block).to(DEV)
        value = torch.nn.functional.one_hot(mark, dim).to(torch.bfloat16).unsqueeze(1).expand(-1, kv_heads, -1).to(DEV)
        hip_ops.paged_kv4_append(torch.zeros_like(value), value, *pools, slots, block)
    return tables.to(DEV), pools, [m.to(DEV) for m in marks]


def _shares(got, mark, length, dim):
    """``got`` (heads, D): with all scores 0 each probability is 1, exact in bf16, and dim d gets its count over ``length``:
    one rounding to bf16 (2^-8), a division and a product in 32 bits (2^-22).  Tokens of one mark that were lost or counted
    twice would move their dim's share by more than twice that."""
    count = torch.bincount(mark[:length], minlength=dim).double()
    lost = _together(len(mark))
    assert length <= 2 * lost or lost / count.max() - lost / length > 2 * 2.0**-8
    want = count / length
    assert ((got.double() - want).abs() <= (2.0**-8 + 2.0**-22) * want).all(), ((got.double() - want).abs() / want.clamp(min=1e-9)).max().item()


@pytest.mark.parametrize("lens,heads,kv_heads,dim,block", [
    ([70_001], 16, 2, 256, 16), ([140_000, 3], 8, 1, 128, 128), ([200_003], 16, 1, 128, 16), ([4001, 1025, 7, 2500], 16, 2, 256, 16), ([1100] * 30 + [5000], 20, 4, 128, 32),
    ([3001], 16, 1, 256, 64), ([12_345, 1, 1024, 33], 9, 1, 128, 16),
])
def test_every_token_of_a_long_row_counts_once_in_decode(lens, heads, kv_heads, dim, block) -> None:
    tables, pools, marks = _marked(lens, kv_heads, dim, block, len(lens) + dim)
    query = torch.zeros(len(lens), heads, 1, dim, dtype=torch.bfloat16, device=DEV)
    got = hip_ops.paged_attention_decode_kv4(query, tables, *pools, torch.tensor(lens, dtype=torch.int32, device=DEV), block)
    for row, n in enumerate(lens):
        _shares(got[row, :, 0], marks[row], n, dim)


@pytest.mark.parametrize("new,prefix,heads,kv_heads,dim,block", [
    ([333], [66_000], 4, 1, 128, 16), ([16], [30_000], 16, 2, 256, 16), ([1], [5000], 16, 2, 256, 64), ([200, 3], [9000, 2001], 20, 4, 128, 32), ([600], [3000], 16, 2, 256, 16),
])
def test_every_token_of_a_long_row_counts_once_in_prefill(new, prefix, heads, kv_heads, dim, block) -> None:
    totals = [n + p for n, p in zip(new, prefix)]
    tables, pools, marks = _marked(totals, kv_heads, dim, block, sum(new) + dim)
    query = torch.zeros(sum(new), heads, dim, dtype=torch.bfloat16, device=DEV)
    cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=DEV)
    got = hip_ops.paged_attention_prefill_kv4(query, cu, torch.tensor(prefix, dtype=torch.int32, device=DEV), *pools, tables, block, max_new=max(new))
    at = 0
    for row, (n, p) in enumerate(zip(new, prefix)):
        for i in sorted({0, n // 2, n - 1, *range(0, n, 37)}):
            _shares(got[at + i], marks[row], p + i + 1, dim)
        at += n


# the rows split many ways (n_wgs > 16 row groups: the merge shares a head's dims) and few ways
SPLIT = [([20_000, 5], 16, 2, 256, 16), ([3000, 40, 1500, 9000] * 4, 16, 2, 256, 16), ([30_000], 16, 1, 128, 32), ([2000, 1, 4000] * 5, 20, 4, 128, 16), ([6000, 0, 1100], 9, 1, 128, 16)]


def _case(lens, heads, kv_heads, dim, block, seed=1, index=torch.int32, width=None, poison=True):
    gen = torch.Generator().manual_seed(seed + len(lens) + dim)
    tables, pools = _cache(gen, lens, kv_heads, dim, block, index, width, poison)
    query = torch.randn(len(lens), heads, 1, dim, generator=gen).to(torch.bfloat16).to(DEV)
    return tables, pools, query, torch.tensor(lens, dtype=index, device=DEV)


def _check(got, tables, pools, query, lens, block, scale=None, gate=None):
    for row, n in enumerate(lens):
        if n <= 0:
            assert not got[row].any()
            continue
        k, v, there = _dense(tables, pools, row, n, block)
        want, mass = _attend(query[row].double().transpose(0, 1), k, v, there[None], scale or query.shape[3] ** -0.5)
        _close(got[row].transpose(0, 1), want, mass, None if gate is None else gate[row : row + 1])


@pytest.mark.parametrize("lens,heads,kv_heads,dim,block", SPLIT)
def test_split_rows_with_strided_tensors(lens, heads, kv_heads, dim, block) -> None:
    tables, pools, query, n = _case(lens, heads, kv_heads, dim, block)
    gate = torch.randn(len(lens), heads, dim, device=DEV).to(torch.bfloat16)
    proj = torch.cat((query[:, :, 0], gate), dim=-1)
    out = torch.full_like(query, 5.0)
    got = hip_ops.paged_attention_decode_kv4(proj[..., None, :dim], tables, *pools, n, block, gate=proj[..., dim:], out=out)
    assert got is out
    _check(got, tables, pools, query, lens, block, gate=gate)
    assert torch.equal(got, hip_ops.paged_attention_decode_kv4(query, tables, *pools, n, block, gate=gate.view(len(lens), -1)))


@pytest.mark.parametrize("scale", [8.0, 1e-6])
@pytest.mark.parametrize("lens,heads,kv_heads,dim,block", SPLIT)
def test_split_rows_with_a_scale(lens, heads, kv_heads, dim, block, scale) -> None:
    tables, pools, query, n = _case(lens, heads, kv_heads, dim, block, seed=2)
    _check(hip_ops.paged_attention_decode_kv4(query, tables, *pools, n, block, scale=scale), tables, pools, query, lens, block, scale=scale)


def test_split_rows_end_at_their_tables() -> None:
    tables, pools, query, n = _case([4096, 4096], 16, 2, 256, 16, index=torch.int64)
    want = hip_ops.paged_attention_decode_kv4(query, tables, *pools, n, 16)
    assert torch.equal(want, hip_ops.paged_attention_decode_kv4(query, tables, *pools, torch.tensor([2**40, 5000], device=DEV), 16))


@pytest.mark.parametrize("lens,heads,kv_heads,dim,block", SPLIT)
def test_a_nan_in_a_split_row_shows_where_it_is_seen(lens, heads, kv_heads, dim, block) -> None:
    """A value group with a NaN reaches its 32 dims of its row and KV head; a query with one, and a key, all dims."""
    tables, pools, query, n = _case(lens, heads, kv_heads, dim, block, seed=3, poison=False)
    group = heads // kv_heads
    want = hip_ops.paged_attention_decode_kv4(query, tables, *pools, n, block)
    assert torch.isfinite(want).all()
    one = torch.ones(1, kv_heads, dim, dtype=torch.bfloat16, device=DEV)
    bad = one.clone()
    bad[0, -1, 40] = float("nan")
    for at in (0, lens[0] // 2, lens[0] - 1):
        slot = (tables[0, at // block].long() * block + at % block).reshape(1)
        saved = [p.clone() for p in pools]
        k, v = (x[0, :, at].clone().unsqueeze(0) for x in hip_ops.paged_kv4_gather(*pools, tables[:1].contiguous(), lens[0], block))
        v[0, -1, 40] = float("nan")
        hip_ops.paged_kv4_append(k, v, *pools, slot, block)
        got = hip_ops.paged_attention_decode_kv4(query, tables, *pools, n, block)
        hit = torch.zeros_like(got, dtype=torch.bool)
        hit[0, heads - group :, :, 32:64] = True
        assert torch.equal(got.isnan(), hit) and torch.equal(got[~hit], want[~hit])
        k[0, -1, 3] = float("-inf")
        hip_ops.paged_kv4_append(k, one, *pools, slot, block)
        got = hip_ops.paged_attention_decode_kv4(query, tables, *pools, n, block)
        assert got[0, heads - group :].isnan().all() and torch.isfinite(got[1:]).all() and torch.isfinite(got[0, : heads - group]).all()
        for p, q in zip(pools, saved):
            p.copy_(q)
    query[0, 1, 0, 9], query[0, 3, 0, 5] = float("nan"), float("inf")
    got = hip_ops.paged_attention_decode_kv4(query, tables, *pools, n, block)
    assert got[0, 1].isnan().all() and got[0, 3].isnan().all()
    keep = torch.ones(heads, dtype=torch.bool)
    keep[[1, 3]] = False
    assert torch.equal(got[0][keep], want[0][keep]) and torch.equal(got[1:], want[1:])


@pytest.mark.parametrize("rows,heads,kv_heads,dim,block", [(1, 16, 2, 256, 16), (5, 16, 2, 256, 16), (40, 12, 4, 128, 32), (3, 16, 1, 128, 16)])
def test_a_graph_whose_rows_grow_and_shrink_past_the_split(rows, heads, kv_heads, dim, block) -> None:
    """All short (a workgroup a row group) -> some long (partials) -> none at all -> short again, in the same workspace."""
    full = [6000] + [1500] * (rows - 1)
    tables, pools, query, n = _case(full, heads, kv_heads, dim, block, seed=4, poison=False)
    gate = torch.randn(rows, heads, dim, device=DEV).to(torch.bfloat16)
    call = lambda: hip_ops.paged_attention_decode_kv4(query, tables, *pools, n, block, gate=gate)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    short = [17 + 30 * r for r in range(rows)]
    for lens in (short, full, [0] * rows, short, [1024] * rows, [1025] + short[1:], [6000] + [0] * (rows - 1), [1] * rows, full):
        lens = [min(a, b) for a, b in zip(lens, full)]
        n.copy_(torch.tensor(lens, dtype=torch.int32))
        query.mul_(-1.01)
        want = call()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        _check(out, tables, pools, query, lens, block, gate=gate)
        (torch.ones(64, device=DEV) * 2).sum().item()


def test_two_graphs_of_split_rows_in_turn() -> None:
    """Captured one after the other, replayed in turn and behind each other."""
    runs = []
    for lens, heads, kv_heads, dim, block in SPLIT[:3]:
        tables, pools, query, n = _case(lens, heads, kv_heads, dim, block, seed=5)
        call = lambda t=tables, p=pools, q=query, n=n, b=block: hip_ops.paged_attention_decode_kv4(q, t, *p, n, b)  # noqa: E731
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        runs.append((query, call, graph, out))
    for _ in range(3):
        for query, _, _, _ in runs:
            query.mul_(-1.01)
        for _, _, graph, _ in runs:
            graph.replay()
        torch.cuda.synchronize()
        for _, call, _, out in runs:
            assert torch.equal(out, call())


@pytest.mark.parametrize("lens,heads,kv_heads,dim,block", SPLIT[:2])
def test_split_rows_on_another_stream(lens, heads, kv_heads, dim, block) -> None:
    tables, pools, query, n = _case(lens, heads, kv_heads, dim, block, seed=6)
    want = hip_ops.paged_attention_decode_kv4(query, tables, *pools, n, block)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [hip_ops.paged_attention_decode_kv4(query, tables, *pools, n, block) for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(x, want) for x in got)


@pytest.mark.parametrize("block", [256, 512, 1024])
@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 2, 256), (20, 4, 128)])
def test_large_blocks(block, heads, kv_heads, dim) -> None:
    """Append, gather, plan, prologue, decode and prefill with blocks of up to 1024 tokens, rows that end inside one."""
    lens = [block - 1, block, block + 1, 1, 3 * block - 100]
    gen = torch.Generator().manual_seed(block + dim)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    blocks = sum(-(-x // block) for x in lens) + 2
    pools = [torch.full((blocks, kv_heads, hip_ops.kv4_tile_bytes(dim, block)), 255, dtype=torch.uint8, device=DEV) for _ in range(2)]
    tables, n = torch.full((len(lens), 5), -1, dtype=torch.int32, device=DEV), i32([0] * len(lens))
    free, state, status = torch.arange(blocks, dtype=torch.int32, device=DEV), i32([0, blocks]), i32([9])
    plan = hip_ops.paged_kv_plan(tables, n, i32(lens), free, state, status, block, max_tokens=sum(lens))
    assert int(status) == 0 and n.tolist() == lens
    q, k, v = (torch.randn(sum(lens), h, d, generator=gen).to(torch.bfloat16).to(DEV) for h, d in ((heads, 2 * dim), (kv_heads, dim), (kv_heads, dim)))
    w = torch.zeros(dim, dtype=torch.bfloat16, device=DEV)
    query, gate = hip_ops.qk_norm_mrope_kv_append(q, k, v, w, w, plan.positions, (dim // 8,), *pools, plan.slots, block, eps=1e-6, rope_theta=1e6)
    small = [torch.zeros(-(-sum(lens) // 16), kv_heads, 16, dim, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    hip_ops.qk_norm_mrope_kv_append(q, k, v, w, w, plan.positions, (dim // 8,), *small, torch.arange(sum(lens), device=DEV), 16, eps=1e-6, rope_theta=1e6)
    dense = [x.transpose(1, 2).reshape(-1, kv_heads, dim)[: sum(lens)] for x in small]
    again = [torch.full_like(p, 255) for p in pools]
    hip_ops.paged_kv4_append(*dense, *again, plan.slots, block)
    assert torch.equal(pools[0], again[0]) and torch.equal(pools[1], again[1])
    flat = [torch.zeros(-(-sum(lens) // 16), kv_heads, hip_ops.kv4_tile_bytes(dim, 16), dtype=torch.uint8, device=DEV) for _ in range(2)]
    hip_ops.paged_kv4_append(*dense, *flat, torch.arange(sum(lens), device=DEV), 16)
    want = hip_ops.paged_kv4_gather(*flat, torch.arange(flat[0].shape[0], dtype=torch.int32, device=DEV), sum(lens), 16)
    prefill = hip_ops.paged_attention_prefill_kv4(query, plan.cu_seqlens, plan.starts, *pools, tables, block, max_new=max(lens), gate=gate)
    last = plan.cu_seqlens[1:].long() - 1
    decode = hip_ops.paged_attention_decode_kv4(query[last].unsqueeze(2), tables, *pools, n, block, gate=gate[last])
    at = 0
    for row, length in enumerate(lens):
        got = hip_ops.paged_kv4_gather(*pools, tables[row : row + 1], length, block)
        keys, values = (x[:, :, at : at + length] for x in want)
        assert torch.equal(got[0], keys) and torch.equal(got[1], values)
        t = torch.arange(length, device=DEV)
        out, mass = _attend(query[at : at + length].double(), keys[0].double(), values[0].double(), t[None] <= t[:, None], dim**-0.5)
        _close(prefill[at : at + length], out, mass, gate[at : at + length])
        _close(decode[row].transpose(0, 1), out[-1:], mass[-1:], gate[at + length - 1 : at + length])
        at += length
