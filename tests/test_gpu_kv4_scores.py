"""Scores whose small products stand beside one large product of the same eight dims: the matrix instruction adds the
eight in fixed point, so the small ones count only by how the query is split."""

from __future__ import annotations

import pytest
import torch

import hip_ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dim,heads,kv_heads", [(256, 16, 2), (128, 9, 1), (256, 3, 1)])
@pytest.mark.parametrize("at", [0, 40, 120])
@pytest.mark.parametrize("tokens", [64, 5000])
def test_small_products_beside_a_large_one(dim, heads, kv_heads, at, tokens) -> None:
    """The large product is the same for every token, 128 * 6, and leaves the softmax alone.  Seven elements of 15/256
    turn it by codes of up to 1, each product below 2^-13 of the large one.  Scores are below 2^13 in units of log 2: their
    sum (768, rounded by up to 2^-14) and its product with the scale 4 / log 2 (up to 2^-11) move a probability by less
    than 2^-9; the rest is the rounding of probabilities and result to bf16."""
    gen = torch.Generator().manual_seed(at + tokens)
    block, scale, small = 16, 4.0, 15 / 256
    codes = torch.randint(-2, 3, (tokens, 7), generator=gen).double() / 2
    signs = torch.randint(0, 2, (heads, 7), generator=gen).double() * 2 - 1
    key = torch.zeros(tokens, kv_heads, dim)
    key[:, :, at] = 6.0
    key[:, :, at + 1 : at + 8] = codes.float().unsqueeze(1)
    score = scale * small * (codes @ signs.T)  # (tokens, heads), without the common part
    value = torch.zeros(tokens, kv_heads, dim)
    for h in range(min(heads, 8)):  # dim h: the tokens that head h prefers (heads past 8 a group share them)
        for g in range(kv_heads):
            value[:, g, h] = (score[:, (g * heads // kv_heads + h) % heads] > 0).float()
    blocks = -(-tokens // block)
    pools = [torch.zeros(blocks, kv_heads, hip_ops.kv4_tile_bytes(dim, block), dtype=torch.uint8, device=DEV) for _ in range(2)]
    hip_ops.paged_kv4_append(key.to(DEV), value.to(DEV), *pools, torch.arange(tokens, device=DEV), block)
    held = hip_ops.paged_kv4_gather(*pools, torch.arange(blocks, dtype=torch.int32, device=DEV), tokens, block)
    assert torch.equal(held[0][0].transpose(0, 1).float().cpu(), key) and torch.equal(held[1][0].transpose(0, 1).float().cpu(), value)
    query = torch.zeros(1, heads, 1, dim)
    query[0, :, 0, at] = 128.0
    query[0, :, 0, at + 1 : at + 8] = (small * signs).float()
    query = query.to(torch.bfloat16).to(DEV)
    tables = torch.arange(blocks, dtype=torch.int32, device=DEV).unsqueeze(0)
    p = torch.softmax(score, 0)
    want = torch.stack([p[:, h] @ value[:, h * kv_heads // heads].double() for h in range(heads)])
    plain = torch.stack([value[:, h * kv_heads // heads].double().mean(0) for h in range(heads)])
    assert (want - plain).abs().max() > 0.05  # what it would be without the small products
    decode = hip_ops.paged_attention_decode_kv4(query, tables, *pools, torch.tensor([tokens], device=DEV), block, scale=scale)[0, :, 0]
    prefill = hip_ops.paged_attention_prefill_kv4(query[:, :, 0], torch.tensor([0, 1], device=DEV), torch.tensor([tokens - 1], device=DEV), *pools, tables, block, max_new=1, scale=scale)[0]
    for got in (decode, prefill):
        assert ((got.double().cpu() - want).abs() <= (2.0**-7 + 2.0**-9) * want).all(), ((got.double().cpu() - want).abs() / want.clamp(min=1e-9)).max()
