"""The prologue with positions of several axes against its formula in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import hip_ops
from oracle import kv4

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 1e-6


def _inputs(seed, tokens, heads, kv_heads, dim, axes, top, gated=True):
    gen = torch.Generator().manual_seed(seed)
    bf = lambda *shape: torch.randn(*shape, generator=gen).to(torch.bfloat16)  # noqa: E731
    q, k, v = bf(tokens, heads, 2 * dim if gated else dim), bf(tokens, kv_heads, dim) * 3, bf(tokens, kv_heads, dim)
    positions = torch.randint(0, top, (axes, tokens), generator=gen)
    return q, k, v, bf(dim) * 0.3, bf(dim) * 0.3, positions


def _close(got, want):
    """One rounding to bf16 (2^-8 of the value) after fp32 arithmetic: the norm's sum, reciprocal root and three products
    (2^-20 of the head's largest element), angles to 2^-24 of a turn and v_sin / v_cos (together 2^-20)."""
    got, want = got.double().cpu().numpy(), np.asarray(want)
    top = np.abs(want).max(-1, keepdims=True)
    bad = np.abs(got - want) > 2.0**-8 * np.abs(want) + 2.0**-18 * top
    assert not bad.any(), (np.abs(got - want)[bad].max(), int(bad.sum()))


SHAPES = [
    (16, 2, 256, (11, 11, 10), True, 1000), (16, 4, 128, (16, 24, 24), False, 300), (8, 8, 128, (16, 8, 8), True, 3_000_000), (3, 1, 256, (32,), False, 200_000),
    (20, 4, 128, (3, 0, 4, 9), False, 50), (2, 1, 64, (8, 8), True, 70_000), (40, 2, 256, (128,), True, 10), (4, 2, 128, (2, 0), True, 9),
]


@pytest.mark.parametrize("heads,kv_heads,dim,sections,interleaved,top", SHAPES)
@pytest.mark.parametrize("tokens,gated,index", [(1, True, torch.int32), (37, False, torch.int64)])
def test_prologue_into_a_bf16_pool(heads, kv_heads, dim, sections, interleaved, top, tokens, gated, index) -> None:
    q, k, v, qw, kw, positions = _inputs(heads + tokens, tokens, heads, kv_heads, dim, len(sections), top, gated)
    block, blocks = 16, tokens // 16 + 3
    slots = torch.randperm(blocks * block)[:tokens]
    if tokens > 3:
        slots[1], slots[2] = -1, blocks * block
    pools = [torch.full((blocks, kv_heads, block, dim), 9.0, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    weights = [w.to(DEV) if gated else w.float().to(DEV) for w in (qw, kw)]
    query, gate = hip_ops.qk_norm_mrope_kv_append(q.to(DEV), k.to(DEV), v.to(DEV), *weights, positions.to(index).to(DEV), sections, *pools, slots.to(index).to(DEV), block, eps=EPS,
                                                  rope_theta=1e7, interleaved=interleaved)
    form = lambda x, w: kv4.norm_mrope(x.double().numpy(), w.double().numpy(), positions.numpy(), sections, interleaved, 1e7, EPS)  # noqa: E731
    _close(query, form(q[..., :dim], qw))
    if gated:
        assert torch.equal(gate.cpu(), q[..., dim:])
    else:
        assert gate is None
    live = [n for n in range(tokens) if 0 <= slots[n] < blocks * block]
    keys, values = (p.transpose(1, 2).reshape(blocks * block, kv_heads, dim).cpu() for p in pools)
    _close(keys[slots[live]], form(k, kw)[live])
    assert torch.equal(values[slots[live]], v[live])
    rest = torch.ones(blocks * block, dtype=torch.bool)
    rest[slots[live]] = False
    assert (keys[rest] == 9).all() and (values[rest] == 9).all()


@pytest.mark.parametrize("heads,kv_heads,dim,sections,block", [(16, 2, 256, (11, 11, 10), 16), (8, 4, 128, (16, 24, 24), 32), (5, 5, 128, (8,), 64), (4, 2, 256, (4,), 32), (6, 3, 128, (2, 4), 16)])
@pytest.mark.parametrize("tokens", [1, 50])
def test_a_4_bit_pool_holds_the_4_bit_form_of_the_bf16_one(heads, kv_heads, dim, sections, block, tokens) -> None:
    q, k, v, qw, kw, positions = (x.to(DEV) for x in _inputs(7, tokens, heads, kv_heads, dim, len(sections), 5000))
    if tokens > 1:
        v[3, 0, 5] = float("inf")
        k[4, 0, 5] = float("nan")
        v[5] = 0
    blocks = tokens // block + 2
    slots = torch.randperm(blocks * block, device=DEV)[:tokens]
    bf = [torch.zeros(blocks, kv_heads, block, dim, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    four, want = ([torch.zeros(blocks, kv_heads, hip_ops.kv4_tile_bytes(dim, block), dtype=torch.uint8, device=DEV) for _ in range(2)] for _ in range(2))
    call = lambda pools: hip_ops.qk_norm_mrope_kv_append(q, k, v, qw, kw, positions, sections, *pools, slots, block, eps=EPS, rope_theta=1e6)  # noqa: E731
    a, b = call(bf), call(four)
    assert torch.equal(a[0], b[0])
    flat = [p.transpose(1, 2).reshape(blocks * block, kv_heads, dim)[slots] for p in bf]
    hip_ops.paged_kv4_append(*flat, *want, slots, block)
    assert torch.equal(four[0], want[0]) and torch.equal(four[1], want[1])


def test_one_axis_is_the_embedding_of_the_plain_prologue() -> None:
    """The plain prologue rounds to bf16 between its steps: the norm, cos and sin, both products and the sum, so up to
    five half steps of 2^-8 on numbers no larger than the head's largest element."""
    tokens, heads, kv_heads, dim, block = 40, 16, 2, 256, 16
    q, k, v, qw, kw, _ = (x.to(DEV) for x in _inputs(9, tokens, heads, kv_heads, dim, 1, 10))
    pools = [[torch.zeros(4, kv_heads, block, dim, dtype=torch.bfloat16, device=DEV) for _ in range(2)] for _ in range(2)]
    start = 77
    tables = torch.full((1, 9), -1, dtype=torch.int32, device=DEV)
    tables[0, 4:9] = torch.tensor([2, 0, 3, 1, -1])  # positions 77 .. 116 are logical blocks 4 .. 7
    at = torch.arange(start, start + tokens, device=DEV)
    slots = tables[0].long()[at // block] * block + at % block
    old, _ = hip_ops.qk_norm_rope_kv_append(q, k, v, qw, kw, *pools[0], tables, torch.tensor([0, tokens], device=DEV, dtype=torch.int32), torch.tensor([start], device=DEV, dtype=torch.int32),
                                            block, max_new=tokens, eps=EPS, rope_theta=1e7, partial_rotary_factor=0.25)
    new, _ = hip_ops.qk_norm_mrope_kv_append(q, k, v, qw, kw, at.expand(3, tokens), (11, 11, 10), *pools[1], slots, block, eps=EPS, rope_theta=1e7, interleaved=True)
    for a, b in ((old, new), (pools[0][0], pools[1][0])):
        top = b.float().abs().amax(-1, keepdim=True)
        assert ((a.float() - b.float()).abs() <= 5 * 2.0**-8 * top).all()
    assert torch.equal(pools[0][1], pools[1][1])


def test_flat_projections_strided_positions_and_refusals() -> None:
    tokens, heads, kv_heads, dim, block = 9, 4, 2, 128, 16
    q, k, v, qw, kw, positions = (x.to(DEV) for x in _inputs(11, tokens, heads, kv_heads, dim, 3, 99))
    pools = [torch.zeros(1, kv_heads, block, dim, dtype=torch.bfloat16, device=DEV) for _ in range(4)]
    slots = torch.arange(tokens, device=DEV)
    kw_args = dict(eps=EPS, rope_theta=1e6)
    a, _ = hip_ops.qk_norm_mrope_kv_append(q, k, v, qw, kw, positions, (4, 4, 4), *pools[:2], slots, block, **kw_args)
    by_token = positions.T.contiguous()
    b, _ = hip_ops.qk_norm_mrope_kv_append(q.view(tokens, -1), k.view(tokens, -1), v.view(tokens, -1), qw, kw, by_token.T, (4, 4, 4), *pools[2:], slots, block, **kw_args)
    assert torch.equal(a, b) and torch.equal(pools[0], pools[2])
    good = [q, k, v, qw, kw, positions, (4, 4, 4), pools[0], pools[1], slots, block]
    for at, bad in ((0, q.float()), (0, q[..., :100]), (1, k[:, :1]), (3, qw[:5]), (3, qw.float()), (5, positions[:2]), (5, positions.float()), (6, (4, 4, 3, 9, 9)), (6, (300, 1, 1)),
                    (6, (1, 1, 1)), (7, pools[0].float()), (9, slots[:3]), (9, slots.float()), (10, 32)):
        args = list(good)
        args[at] = bad
        with pytest.raises(RuntimeError):
            hip_ops.qk_norm_mrope_kv_append(*args, **kw_args)


def test_rotary_dims_that_lanes_would_share_are_refused() -> None:
    q, k, v, qw, kw, positions = (x.to(DEV) for x in _inputs(12, 3, 2, 1, 128, 1, 9))
    pools = [torch.zeros(1, 1, 16, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    with pytest.raises(RuntimeError, match="multiple of 4"):
        hip_ops.qk_norm_mrope_kv_append(q, k, v, qw, kw, positions, (7,), *pools, torch.arange(3, device=DEV), 16, eps=EPS, rope_theta=1e6)


@pytest.mark.parametrize("dim,sections,tokens", [(256, (11, 11, 10), 33), (128, (16, 24, 24), 33), (128, (4, 4), 2050), (256, (16,), 2047), (256, (40, 56), 5)])
def test_rows_of_any_alignment_and_count_agree(dim, sections, tokens) -> None:
    """The same call with every row on 16 bytes and with rows 4 elements off: to a rounding, as the sums run in other orders."""
    heads, kv_heads, block = 6, 2, 16
    q, k, v, qw, kw, positions = (x.to(DEV) for x in _inputs(13, tokens, heads, kv_heads, dim, len(sections), 4000))
    wide = torch.zeros(tokens, (2 * heads + 2 * kv_heads) * dim + 4, dtype=torch.bfloat16, device=DEV)
    parts = [wide[:, 4 + a * dim:4 + b * dim] for a, b in ((0, 2 * heads), (2 * heads, 2 * heads + kv_heads), (2 * heads + kv_heads, 2 * heads + 2 * kv_heads))]
    for part, x in zip(parts, (q, k, v)):
        part.copy_(x.reshape(tokens, -1))
    blocks = tokens // block + 1
    slots = torch.randperm(blocks * block, device=DEV)[:tokens]
    runs = []
    for rows in ((q, k, v), parts):
        pools = [torch.zeros(blocks, kv_heads, block, dim, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
        query, _ = hip_ops.qk_norm_mrope_kv_append(*rows, qw, kw, positions, sections, *pools, slots, block, eps=EPS, rope_theta=1e6)
        runs.append((query, *pools))
    form = kv4.norm_mrope(q[..., :dim].double().cpu().numpy(), qw.double().cpu().numpy(), positions.cpu().numpy(), sections, False, 1e6, EPS)
    for query, keys, values in runs:
        _close(query, form)
        assert torch.equal(values, runs[0][2])
        top = runs[0][1].float().abs().amax(-1, keepdim=True)
        assert ((keys.float() - runs[0][1].float()).abs() <= 2.0**-7 * runs[0][1].float().abs() + 2.0**-17 * top).all()


@pytest.mark.parametrize("shift", [0, 4])
def test_an_infinity_stays_in_its_pair(shift) -> None:
    """x rsqrt(inf) is 0 at every finite x and NaN at the infinity; the rotation mixes a dim with its pair only."""
    dim, sections = 256, (11, 11, 10)
    q, k, v, qw, kw, positions = (x.to(DEV) for x in _inputs(15, 3, 2, 1, dim, 3, 50))
    wide = torch.zeros(3, 4 * dim + shift, dtype=torch.bfloat16, device=DEV)
    rows = wide[:, shift:]
    rows.copy_(q.reshape(3, -1))
    rows[1, 33], rows[2, 2 * dim + 200] = float("inf"), float("inf")  # head 0's dim 33 turns with dim 1; head 1's dim 200 does not turn
    pools = [torch.zeros(1, 1, 16, dim, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    query, _ = hip_ops.qk_norm_mrope_kv_append(rows, k, v, qw, kw, positions, sections, *pools, torch.arange(3, device=DEV), 16, eps=EPS, rope_theta=1e6, interleaved=True)
    assert query[1, 0].isnan().nonzero().flatten().tolist() == [1, 33] and query[2, 1].isnan().nonzero().flatten().tolist() == [200]
    assert (query[1, 0].nan_to_num() == 0).all() and (query[2, 1].nan_to_num() == 0).all() and query.isnan().sum() == 3
