"""Workspace of the prefill over the 4-bit cache: bounded by the tokens that can be computed, not by padding."""

from __future__ import annotations

import random

import hip_loader as L


def _bytes(total, batch, max_new, heads, kv_heads, dim, tokens) -> int:
    return L.load_library().qa_paged_attention_prefill_kv4_workspace(total, batch, max_new, heads, kv_heads, dim, tokens)


def test_a_padded_query_asks_for_no_more_than_its_rows_can_fill() -> None:
    rng = random.Random(0)
    split = 0
    for _ in range(3000):
        kv_heads, dim = rng.choice((1, 2, 4, 8)), rng.choice((128, 256))
        heads = kv_heads * rng.randint(1, 16)
        batch, max_new, tokens = rng.randint(1, 40), int(2 ** rng.uniform(0, 11)), int(2 ** rng.uniform(5, 20))
        fit = _bytes(batch * max_new, batch, max_new, heads, kv_heads, dim, tokens)
        split += fit > 0
        # a column tile of 128 for every workgroup, at most 256 of them, of dim sums and two statistics
        assert fit <= 256 * 128 * (dim + 2) * 4
        for total in (batch * max_new + 1, batch * max_new + 5000, 2**20):
            assert _bytes(total, batch, max_new, heads, kv_heads, dim, tokens) == fit
    assert split > 1000


def test_one_row_of_sixteen_tokens_in_a_step_of_8192() -> None:
    assert _bytes(8192, 1, 16, 16, 2, 256, 32768) == _bytes(16, 1, 16, 16, 2, 256, 32768) > 0
