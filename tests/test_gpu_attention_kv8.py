"""Attention over the 8-bit cache against softmax attention in 64 bits on the values the cache holds."""

from __future__ import annotations

import random

import pytest
import torch

import hip_ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _cache(gen, totals, kv_heads, dim, block, index=torch.int32, width=None, poison=True):
    """An 8-bit pool with the rows' blocks in random order; slots past a row's end hold NaNs where poison."""
    need = [-(-n // block) for n in totals]
    blocks = sum(need) + 3
    order = torch.randperm(blocks, generator=gen)
    tables = torch.full((len(totals), max(max(need), width or 1)), -1, dtype=index)
    at = 0
    for row, n in enumerate(need):
        tables[row, :n] = order[at : at + n].to(index)
        at += n
    pools = [torch.zeros(blocks, kv_heads, hip_ops.kv8_tile_bytes(dim, block), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2)]
    n = blocks * block
    x = torch.randn(2, n, kv_heads, dim, generator=gen)
    x[0] *= torch.exp(0.5 * torch.randn(kv_heads, dim, generator=gen))
    if poison:
        used = torch.zeros(n, dtype=torch.bool)
        for row, total in enumerate(totals):
            t = torch.arange(total)
            used[tables[row].long()[t // block] * block + t % block] = True
        x[:, ~used] = float("nan")
    hip_ops.paged_kv8_append(x[0].to(DEV), x[1].to(DEV), *pools, torch.arange(n, device=DEV), block)
    return tables.to(DEV), pools


def _dense(tables, pools, row, length, block):
    """Keys, values (kv_heads, length, D) in 64 bits and whether each token is there."""
    k, v = hip_ops.paged_kv8_gather(*pools, tables[row : row + 1].contiguous(), length, block)
    ids = tables[row].long()[: -(-length // block)].repeat_interleave(block)[:length]
    return k[0].double(), v[0].double(), (ids >= 0) & (ids < pools[0].shape[0])


def _attend(q, k, v, seen, scale):
    """q (n, heads, D), k/v (kv_heads, T, D), seen (n, T): the result and sum_t p_t |v_t|."""
    group = q.shape[1] // k.shape[0]
    out, mass = torch.zeros_like(q), torch.zeros_like(q)
    any_seen = seen.any(-1)
    keep = seen.any(0)
    k, v, seen = k[:, keep].contiguous(), v[:, keep].contiguous(), seen[:, keep]
    for h in range(q.shape[1]):
        s = (q[:, h] @ k[h // group].T.contiguous() * scale).masked_fill(~seen, -torch.inf)
        p = torch.softmax(s[any_seen], -1)
        out[any_seen, h] = p @ v[h // group]
        mass[any_seen, h] = p @ v[h // group].abs()
    return out, mass


def _close(got, want, mass, gate=None):
    """bf16 rounds the result (2^-8 of it) and each probability (2^-8 of sum p |v|); scores, exponentials and sums in 32
    bits are within 2^-12 of that sum."""
    if gate is not None:
        s = torch.sigmoid(gate.double())
        want, mass = want * s, mass * s
    err = (got.double() - want).abs()
    bound = 2.0**-8 * (want.abs() + mass) + 2.0**-12 * mass + 1e-30
    assert torch.isfinite(got).all()
    assert (err <= bound).all(), (err / bound).max().item()


def _check_decode(seed, lens, heads, kv_heads, dim, block, index=torch.int32, gated=False, width=None, holes=False, scale=None):
    gen = torch.Generator().manual_seed(seed)
    tables, pools = _cache(gen, [max(n, 0) for n in lens], kv_heads, dim, block, index, width)
    if holes:
        tables[:, 0] = -1
        if tables.shape[1] > 3:
            tables[0, 2] = pools[0].shape[0]
    query = torch.randn(len(lens), heads, 1, dim, generator=gen).to(torch.bfloat16).to(DEV)
    gate = torch.randn(len(lens), heads, dim, generator=gen).to(torch.bfloat16).to(DEV) if gated else None
    got = hip_ops.paged_attention_decode_kv8(query, tables, *pools, torch.tensor(lens, dtype=index, device=DEV), block, gate=gate, scale=scale)
    assert got.shape == query.shape
    for row, n in enumerate(lens):
        if n <= 0:
            assert not got[row].any()
            continue
        k, v, there = _dense(tables, pools, row, min(n, tables.shape[1] * block), block)
        want, mass = _attend(query[row].double().transpose(0, 1), k, v, there[None], scale or dim**-0.5)
        _close(got[row].transpose(0, 1), want, mass, None if gate is None else gate[row : row + 1])
    return query, tables, pools, got


GROUPS = [(16, 2, 256), (16, 1, 256), (8, 8, 128), (6, 2, 256), (16, 1, 128), (9, 1, 128), (20, 4, 128), (3, 1, 256), (12, 4, 128)]


@pytest.mark.parametrize("heads,kv_heads,dim", GROUPS)
@pytest.mark.parametrize("block", [16, 64])
def test_decode_of_every_group_size(heads, kv_heads, dim, block) -> None:
    _check_decode(heads * dim + block, [1, 15, 16, 17, 0, 31, 32, 33, 64, 65, 257, -3, 700], heads, kv_heads, dim, block, gated=block == 64)


@pytest.mark.parametrize("index,width", [(torch.int64, None), (torch.int32, 400)])
def test_decode_with_wide_tables_and_holes(index, width) -> None:
    _check_decode(3, [40, 300, 16, 1000], 16, 2, 256, 16, index, True, width, holes=True)
    _check_decode(4, [40, 300, 33, 1000], 16, 1, 128, 32, index, True, width, holes=True)


def test_decode_of_one_long_row_and_of_many_short_ones() -> None:
    _check_decode(5, [70_001], 16, 2, 256, 16)
    _check_decode(6, [140_000, 3], 8, 1, 128, 128, torch.int64)
    rng = random.Random(0)
    _check_decode(7, [rng.randint(0, 90) for _ in range(200)], 16, 2, 256, 16, gated=True)
    _check_decode(8, [rng.choice((1, 2000, 9000)) for _ in range(40)], 8, 2, 128, 16)


def test_decode_lengths_past_the_table_stop_at_it() -> None:
    gen = torch.Generator().manual_seed(9)
    tables, pools = _cache(gen, [64, 64], 2, 256, 16)
    query = torch.randn(2, 16, 1, 256, generator=gen).to(torch.bfloat16).to(DEV)
    at, past = (hip_ops.paged_attention_decode_kv8(query, tables, *pools, torch.tensor(n, device=DEV), 16) for n in ([64, 64], [1000, 2**40]))
    assert torch.equal(at, past)


def test_decode_reads_strided_queries_and_gates_and_writes_out() -> None:
    query, tables, pools, want = _check_decode(10, [50, 300, 7], 16, 2, 256, 16)
    lens = torch.tensor([50, 300, 7], device=DEV, dtype=torch.int32)
    proj = torch.randn(3, 16, 512, device=DEV).to(torch.bfloat16)
    proj[..., :256] = query[:, :, 0]
    out = torch.full_like(query, 5.0)
    got = hip_ops.paged_attention_decode_kv8(proj[..., None, :256], tables, *pools, lens, 16, out=out)
    assert got is out and torch.equal(out, want)
    gated = hip_ops.paged_attention_decode_kv8(query, tables, *pools, lens, 16, gate=proj[..., 256:])
    flat = hip_ops.paged_attention_decode_kv8(query, tables, *pools, lens, 16, gate=proj[..., 256:].reshape(3, -1))
    assert torch.equal(gated, flat) and not torch.equal(gated, want)


def test_decode_with_scores_far_apart_and_a_scale() -> None:
    """Scores in the hundreds: all of the mass on one token, the others underflow."""
    _check_decode(11, [300, 40], 16, 2, 256, 16, scale=8.0)
    _check_decode(12, [300, 40], 16, 2, 256, 16, scale=1e-6)


def test_a_nan_in_a_visible_value_or_query_shows() -> None:
    gen = torch.Generator().manual_seed(13)
    tables, pools = _cache(gen, [40, 40], 1, 256, 16, poison=False)
    query = torch.randn(2, 8, 1, 256, generator=gen).to(torch.bfloat16).to(DEV)
    query[0, 3, 0, 9] = float("nan")
    query[0, 5, 0, 9] = float("inf")
    lens = torch.tensor([40, 40], device=DEV)
    slots = tables[1, 1].long() * 16 + torch.arange(16, device=DEV)
    fine = torch.ones(16, 1, 256, dtype=torch.bfloat16, device=DEV)
    bad = fine.clone()
    bad[3, 0, 40] = float("nan")
    got = hip_ops.paged_attention_decode_kv8(query, tables, *pools, lens, 16)
    assert got[0, 3].isnan().all() and got[0, 5].isnan().all() and torch.isfinite(got[0, :3]).all() and torch.isfinite(got[1]).all()
    hip_ops.paged_kv8_append(fine, bad, *pools, slots, 16)
    got = hip_ops.paged_attention_decode_kv8(query, tables, *pools, lens, 16)
    assert got[1, :, :, 40].isnan().all() and torch.isfinite(got[1, :, :, :40]).all() and torch.isfinite(got[1, :, :, 41:]).all()  # a value: its dim only
    hip_ops.paged_kv8_append(bad, fine, *pools, slots, 16)
    got = hip_ops.paged_attention_decode_kv8(query, tables, *pools, lens, 16)
    assert got[1].isnan().all()  # a key: every dim


def test_captured_decode_replays_as_eager_runs() -> None:
    gen = torch.Generator().manual_seed(14)
    tables, pools = _cache(gen, [600, 600, 600], 2, 256, 16)
    query = torch.randn(3, 16, 1, 256, generator=gen).to(torch.bfloat16).to(DEV)
    lens = torch.tensor([1, 300, 600], device=DEV, dtype=torch.int32)
    call = lambda: hip_ops.paged_attention_decode_kv8(query, tables, *pools, lens, 16)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for step in range(5):
        lens.copy_(torch.tensor([1 + step, 300 - 60 * step, 600 - step]))
        query.mul_(-1.01)
        want = call()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_decode_on_another_stream() -> None:
    query, tables, pools, want = _check_decode(15, [50, 300, 7], 16, 2, 256, 16)
    lens = torch.tensor([50, 300, 7], device=DEV, dtype=torch.int32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = hip_ops.paged_attention_decode_kv8(query, tables, *pools, lens, 16)
    side.synchronize()
    assert torch.equal(got, want)


def test_empty_batch() -> None:
    _, tables, pools, _ = _check_decode(16, [5], 16, 2, 256, 16)
    got = hip_ops.paged_attention_decode_kv8(torch.zeros(0, 16, 1, 256, dtype=torch.bfloat16, device=DEV), tables[:0], *pools, torch.zeros(0, dtype=torch.int32, device=DEV), 16)
    assert got.shape == (0, 16, 1, 256)


# --------------------------------------------------------------------------- prefill


def _check_prefill(seed, new, prefix, heads, kv_heads, dim, block, index=torch.int32, gated=True, holes=False, pad=0, scale=None, width=None):
    gen = torch.Generator().manual_seed(seed)
    tables, pools = _cache(gen, [n + p for n, p in zip(new, prefix)], kv_heads, dim, block, index, width)
    if holes:
        tables[:, 0] = -1
        if tables.shape[1] > 3:
            tables[0, 2] = pools[0].shape[0]
    total = sum(new)
    query = torch.randn(total + pad, heads, dim, generator=gen).to(torch.bfloat16).to(DEV)
    gate = torch.randn(total + pad, heads, dim, generator=gen).to(torch.bfloat16).to(DEV) if gated else None
    cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=index, device=DEV)
    out = torch.full_like(query, 3.0)
    got = hip_ops.paged_attention_prefill_kv8(query, cu, torch.tensor(prefix, dtype=index, device=DEV), *pools, tables, block, max_new=max(new), gate=gate, scale=scale, out=out)
    assert got is out and (got[total:] == 3).all()
    at = 0
    for row, (n, p) in enumerate(zip(new, prefix)):
        if n == 0:
            continue
        k, v, there = _dense(tables, pools, row, n + p, block)
        t = torch.arange(n + p, device=DEV)
        seen = (t[None] <= p + torch.arange(n, device=DEV)[:, None]) & there[None]
        want, mass = _attend(query[at : at + n].double(), k, v, seen, scale or dim**-0.5)
        none = ~seen.any(-1)
        assert not got[at : at + n][none].any()
        _close(got[at : at + n], want, mass, None if gate is None else gate[at : at + n])
        at += n
    return query, cu, tables, pools, got, gate


@pytest.mark.parametrize("heads,kv_heads,dim", GROUPS)
@pytest.mark.parametrize("block", [16, 64])
def test_prefill_of_every_group_size(heads, kv_heads, dim, block) -> None:
    _check_prefill(heads * dim + block, [1, 17, 0, 70, 130], [0, 15, 9, 100, 64], heads, kv_heads, dim, block, gated=block == 16)


@pytest.mark.parametrize("new,prefix", [([1], [0]), ([1], [5000]), ([15, 16, 17, 31, 33], [0, 0, 0, 0, 0]), ([64, 65, 63, 128], [63, 64, 65, 1]), ([300, 1, 2, 0], [3000, 0, 17, 40]), ([900], [0])])
@pytest.mark.parametrize("dim,block", [(256, 16), (128, 32)])
def test_prefill_around_tile_edges(new, prefix, dim, block) -> None:
    _check_prefill(len(new) + dim, new, prefix, 8, 2, dim, block, torch.int64, pad=5)


def test_prefill_with_holes_and_scales() -> None:
    _check_prefill(21, [40, 3, 100], [5, 0, 300], 16, 2, 256, 16, holes=True)
    _check_prefill(22, [40, 3, 100], [5, 0, 300], 16, 1, 128, 16, holes=True, scale=4.0)


def test_prefill_of_many_rows_and_of_a_long_one() -> None:
    rng = random.Random(1)
    _check_prefill(23, [rng.randint(0, 40) for _ in range(150)], [rng.randint(0, 60) for _ in range(150)], 16, 2, 256, 16)
    _check_prefill(24, [333], [66_000], 4, 1, 128, 16)


@pytest.mark.parametrize("new,prefix", [([300, 260, 1, 0, 41], [900, 0, 1200, 7, 64]), ([600], [600]), ([64, 64, 64, 64, 8, 100, 33, 64, 5], [1100, 63, 64, 65, 1, 0, 1000, 0, 15])])
@pytest.mark.parametrize("holes", [False, True])
def test_prefill_of_many_columns_behind_many_keys(new, prefix, holes) -> None:
    """Workgroups of 128 columns, a row's last ones part of them."""
    _check_prefill(29 + len(new), new, prefix, 16, 2, 256, 16, holes=holes, width=100, pad=2)
    _check_prefill(39 + len(new), new, prefix, 16, 1, 256, 64, torch.int64, gated=False, holes=holes, width=30)


def test_prefill_of_one_token_is_decode() -> None:
    query, cu, tables, pools, got, _ = _check_prefill(25, [1, 1, 1], [0, 77, 500], 16, 2, 256, 16, gated=False)
    one = hip_ops.paged_attention_decode_kv8(query.unsqueeze(2), tables, *pools, torch.tensor([1, 78, 501], device=DEV), 16)
    assert ((one[:, :, 0].float() - got.float()).abs() <= 3 * 2.0**-8 * got.float().abs().amax()).all()


def test_prefill_reads_strided_projections() -> None:
    query, cu, tables, pools, want, gate = _check_prefill(26, [30, 9], [4, 60], 16, 2, 256, 16)
    proj = torch.cat((query, gate), dim=-1)
    prefix = torch.tensor([4, 60], dtype=torch.int32, device=DEV)
    got = hip_ops.paged_attention_prefill_kv8(proj[..., :256], cu, prefix, *pools, tables, 16, max_new=30, gate=proj[..., 256:])
    assert torch.equal(got, want)


def test_prefill_with_index_arrays_that_are_off_stays_in_bounds() -> None:
    """cu_seqlens past the query's rows, negative prefixes, a prefix past the table: those tokens are skipped or see what is there."""
    query, cu, tables, pools, want, gate = _check_prefill(27, [30, 9], [4, 60], 16, 2, 256, 16)
    run = lambda c, p: hip_ops.paged_attention_prefill_kv8(query, torch.tensor(c, dtype=torch.int32, device=DEV), torch.tensor(p, dtype=torch.int32, device=DEV), *pools, tables, 16,  # noqa: E731
                                                           max_new=30, gate=gate)
    got = run([0, 30, 2000], [4, 60])
    assert torch.equal(got[:39], want[:39])
    got = run([0, 30, 39], [-1000, 60])
    assert not got[:30].any() and torch.equal(got[30:], want[30:])
    assert torch.isfinite(run([0, 30, 39], [4, 100_000])[:30]).all()


def test_refusals_of_tensors() -> None:
    query, cu, tables, pools, _, gate = _check_prefill(28, [3], [0], 16, 2, 256, 16)
    p = torch.zeros(1, dtype=torch.int32, device=DEV)
    ok = dict(max_new=3)
    for args, kw in (((query.float(), cu, p, *pools, tables, 16), ok), ((query, cu.long(), p, *pools, tables, 16), ok), ((query, cu[:1], p, *pools, tables, 16), ok),
                     ((query[..., :128], cu, p, *pools, tables, 16), ok), ((query[:, :15], cu, p, *pools, tables, 16), ok), ((query, cu, p, *pools, tables, 32), ok),
                     ((query, cu, p, *pools, tables[:0], 16), ok), ((query, cu, p, *pools, tables, 16), dict(max_new=3, gate=gate.float())),
                     ((query, cu, p, *pools, tables, 16), dict(max_new=3, gate=gate[:1])), ((query, cu, p, *pools, tables, 16), dict(max_new=3, out=query.float())),
                     ((query, cu, p, *pools, tables, 16), dict(max_new=-1))):
        with pytest.raises(RuntimeError):
            hip_ops.paged_attention_prefill_kv8(*args, **kw)
    q1 = query[:1].unsqueeze(2)
    for args in ((q1.float(), tables, *pools, p, 16), (q1, tables[:0], *pools, p, 16), (q1, tables, *pools, p.float(), 16), (q1.transpose(1, 2), tables, *pools, p, 16),
                 (q1, tables, *pools, p.repeat(2), 16), (q1, tables.float(), *pools, p, 16), (q1, tables.cpu(), *pools, p, 16), (q1, tables, pools[0], pools[1][:1], p, 16)):
        with pytest.raises(RuntimeError):
            hip_ops.paged_attention_decode_kv8(*args)


@pytest.mark.parametrize("dim,heads,new,prefix,width", [(256, 16, 150, 70, None), (128, 6, 150, 70, None), (256, 16, 550, 70, 80)])
def test_prefill_keeps_a_nan_to_the_tokens_that_see_it(dim, heads, new, prefix, width) -> None:
    gen = torch.Generator().manual_seed(29)
    block = 16
    tables, pools = _cache(gen, [new + prefix], 2, dim, block, width=width)
    query = torch.randn(new, heads, dim, generator=gen).to(torch.bfloat16).to(DEV)
    cu = torch.tensor([0, new], device=DEV)
    run = lambda: hip_ops.paged_attention_prefill_kv8(query, cu, torch.tensor([prefix], device=DEV), *pools, tables, block, max_new=new)  # noqa: E731
    group = heads // 2
    for at in (new + prefix - 1, new + prefix - 25, 130, 70, 30):
        saved = [p.clone() for p in pools]
        run0 = at // 16 * 16
        tokens = torch.arange(run0, min(run0 + 16, new + prefix), device=DEV)
        slots = tables[0, tokens // block].long() * block + tokens % block
        k, v = (x[0, :, tokens].transpose(0, 1).contiguous() for x in hip_ops.paged_kv8_gather(*pools, tables, new + prefix, block))
        # the run written again is the same run: its values are codes already, its largest fits the same scale or a smaller one
        bad = v.clone()
        bad[at - run0, 1, 40] = float("nan")
        hip_ops.paged_kv8_append(k, v, *pools, slots, block)
        base = run()
        hip_ops.paged_kv8_append(k, bad, *pools, slots, block)
        got = run()
        first = max(at - prefix, 0)
        assert torch.equal(got[:first], base[:first])
        assert torch.equal(got[:, :group], base[:, :group])  # the other KV head
        assert got[first:, group:, 40].isnan().all()
        assert torch.equal(got[first:, group:, :40], base[first:, group:, :40]) and torch.equal(got[first:, group:, 41:], base[first:, group:, 41:])
        bad = k.clone()
        bad[at - run0, 1, 3] = float("inf")  # a key: every dim of the tokens that see it
        hip_ops.paged_kv8_append(bad, v, *pools, slots, block)
        got = run()
        assert torch.equal(got[:first], base[:first]) and got[first:, group:].isnan().all() and torch.isfinite(got[:, :group]).all()
        for p, q in zip(pools, saved):
            p.copy_(q)


def test_captured_prefill_replays_as_eager_runs() -> None:
    query, cu, tables, pools, _, gate = _check_prefill(30, [30, 9], [400, 60], 16, 2, 256, 16)
    prefix = torch.tensor([400, 60], dtype=torch.int32, device=DEV)
    call = lambda: hip_ops.paged_attention_prefill_kv8(query, cu, prefix, *pools, tables, 16, max_new=30, gate=gate)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for _ in range(4):
        query.mul_(-1.01)
        prefix.sub_(torch.tensor([7, 1], device=DEV, dtype=torch.int32))
        want = call()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("new,prefix,heads,kv_heads,dim", [([7], [9000], 16, 2, 256), ([40, 3], [3000, 20_000], 8, 2, 128), ([1, 0, 5], [0, 50, 12_000], 16, 1, 256)])
def test_prefill_of_few_tokens_splits_the_keys(new, prefix, heads, kv_heads, dim) -> None:
    _check_prefill(sum(new) + dim, new, prefix, heads, kv_heads, dim, 32, gated=True, holes=dim == 128)


@pytest.mark.parametrize("longest", [1024, 1025, 700])
@pytest.mark.parametrize("rows,heads,kv_heads,dim", [(4, 16, 2, 256), (70, 12, 4, 128), (5, 16, 1, 256)])
@pytest.mark.parametrize("width", [None, 300])
def test_decode_of_short_rows(longest, rows, heads, kv_heads, dim, width) -> None:
    """A workgroup a row group where no row is longer than 1024 tokens, with tables that could hold longer ones and without."""
    rng = random.Random(rows + longest)
    lens = [longest, 0, 1, 33] + [rng.choice((0, 17, rng.randint(1, 300))) for _ in range(rows - 4)]
    _check_decode(21, lens, heads, kv_heads, dim, 16, gated=rows == 4, width=width, holes=rows == 70)


@pytest.mark.parametrize("heads,kv_heads,dim", GROUPS)
def test_decode_of_every_group_size_beside_long_rows(heads, kv_heads, dim) -> None:
    _check_decode(22, [1, 15, 0, 2000, 31, 32, -3, 33, 1100, 16], heads, kv_heads, dim, 16, gated=True)
    _check_decode(23, [3] * 63 + [0, 1500] + [7] * 70, heads, kv_heads, dim, 16)


def test_decode_of_more_row_groups_than_take_a_workgroup_each() -> None:
    """2100 rows of two KV heads: with tables that could hold longer rows they are split over the usual workgroups."""
    rng = random.Random(5)
    lens = [rng.choice((0, 1, 16, 40)) for _ in range(2100)]
    for width in (None, 70):
        _check_decode(24, lens, 4, 2, 128, 16, width=width)


@pytest.mark.parametrize("new,prefix", [([200], [0]), ([3, 16, 40, 0, 1], [0, 5000, 700, 9, 300]), ([130, 2], [400, 0]), ([1], [0])])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 1, 256), (6, 1, 128), (16, 2, 256)])
def test_prefill_with_tables_much_wider_than_the_rows(new, prefix, heads, kv_heads, dim) -> None:
    """The launch has room for many parts; the columns of a row are split by what they see."""
    _check_prefill(26, new, prefix, heads, kv_heads, dim, 16, width=3000, pad=3, holes=kv_heads == 2)


def test_decode_in_one_stream_beside_another() -> None:
    """Two calls at once, each with partial results of its own."""
    cases = [_check_decode(40 + i, [9000 - 100 * i, 40], 16, 2, 256, 16) for i in range(2)]
    lens = [torch.tensor([9000 - 100 * i, 40], dtype=torch.int32, device=DEV) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for _ in range(8):
        for stream, (query, tables, pools, _want), n in zip(streams, cases, lens):
            with torch.cuda.stream(stream):
                got.append(hip_ops.paged_attention_decode_kv8(query, tables, *pools, n, 16))
    torch.cuda.synchronize()
    assert all(torch.equal(out, cases[i % 2][3]) for i, out in enumerate(got))


def test_prefill_in_one_stream_beside_another() -> None:
    """Two calls at once, each with partial results of its own where the keys are split, and one of each number of columns."""
    cases = [(*_check_prefill(60, [20, 3], [6000, 900], 16, 2, 256, 16), [6000, 900], 20), (*_check_prefill(61, [400, 300], [900, 1100], 16, 2, 256, 16), [900, 1100], 400)]
    prefixes = [torch.tensor(case[6], dtype=torch.int32, device=DEV) for case in cases]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for stream, (query, cu, tables, pools, _out, gate, _p, most), prefix in zip(streams, cases, prefixes):
            with torch.cuda.stream(stream):
                got.append(hip_ops.paged_attention_prefill_kv8(query, cu, prefix, *pools, tables, 16, max_new=most, gate=gate))
    torch.cuda.synchronize()
    assert all(torch.equal(out, cases[i % 2][4]) for i, out in enumerate(got))


@pytest.mark.parametrize("dim,kv_heads", [(256, 2), (128, 1)])
def test_pools_past_four_gigabytes(dim, kv_heads) -> None:
    """The last blocks of a pool of 5 GB: offsets do not fit 32 bits."""
    tile = hip_ops.kv8_tile_bytes(dim, 16)
    blocks = 5 * 2**30 // (tile * kv_heads)
    pools = [torch.empty(blocks, kv_heads, tile, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2)]
    gen = torch.Generator().manual_seed(50)
    new, prefix = 20, 300
    total = new + prefix
    need = -(-total // 16)
    tables = torch.stack((torch.arange(blocks - 1, blocks - 1 - need, -1), torch.arange(need))).to(torch.int32).to(DEV)
    x = torch.randn(2, total, kv_heads, dim, generator=gen).to(torch.bfloat16).to(DEV)
    tokens = torch.arange(total, device=DEV)
    for row in range(2):
        hip_ops.paged_kv8_append(x[0], x[1], *pools, tables[row, tokens // 16].long() * 16 + tokens % 16, 16)
    k, v = hip_ops.paged_kv8_gather(*pools, tables, total, 16)
    assert torch.equal(k[0], k[1]) and torch.equal(v[0], v[1])
    query = torch.randn(new, 8, dim, generator=gen).to(torch.bfloat16).to(DEV)
    both = hip_ops.paged_attention_prefill_kv8(torch.cat((query, query)), torch.tensor([0, new, 2 * new], device=DEV), torch.tensor([prefix, prefix], device=DEV), *pools, tables, 16,
                                               max_new=new)
    assert torch.equal(both[:new], both[new:])
    seen = torch.arange(total, device=DEV)[None] <= prefix + torch.arange(new, device=DEV)[:, None]
    want, mass = _attend(query.double(), k[0].double(), v[0].double(), seen, dim**-0.5)
    _close(both[:new], want, mass)
    one = hip_ops.paged_attention_decode_kv8(query[-1:, :, None].expand(2, -1, -1, -1), tables, *pools, torch.tensor([total, total], device=DEV), 16)
    assert torch.equal(one[0], one[1])
    _close(one[:1, :, 0], want[-1:], mass[-1:])


def test_a_query_with_one_element_far_above_the_others() -> None:
    """Its small products count beside the large one: keys are small where the query is large."""
    gen = torch.Generator().manual_seed(51)
    tables, pools = _cache(gen, [400], 1, 256, 16, poison=False)
    x = torch.randn(2, 400, 1, 256, generator=gen)
    x[0, :, :, 7] /= 1000
    tokens = torch.arange(400)
    slots = tables[0].cpu().long()[tokens // 16] * 16 + tokens % 16
    hip_ops.paged_kv8_append(x[0].to(DEV), x[1].to(DEV), *pools, slots.to(DEV), 16)
    query = torch.randn(1, 8, 1, 256, generator=gen)
    query[..., 7] = 300
    query = query.to(torch.bfloat16).to(DEV)
    k, v, there = _dense(tables, pools, 0, 400, 16)
    want, mass = _attend(query[0].double().transpose(0, 1), k, v, there[None], 256**-0.5)
    _close(hip_ops.paged_attention_decode_kv8(query, tables, *pools, torch.tensor([400], device=DEV), 16)[0].transpose(0, 1), want, mass)
    got = hip_ops.paged_attention_prefill_kv8(query[:, :, 0], torch.tensor([0, 1], device=DEV), torch.tensor([399], device=DEV), *pools, tables, 16, max_new=1)
    _close(got, want, mass)
