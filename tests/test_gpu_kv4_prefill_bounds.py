"""Which rows a prefill over the 4-bit cache writes, whatever the tables' width and the query's padding make of the launch."""

from __future__ import annotations

import pytest
import torch

import hip_ops
from test_gpu_attention_kv4 import _attend, _cache, _close, _dense

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _check(seed, new, prefix, max_new, heads, kv_heads, dim, block, width, padded=0, index=torch.int32):
    """Tokens below ``max_new`` of their row against 64 bits, all other rows of ``out`` as they were."""
    gen = torch.Generator().manual_seed(seed)
    tables, pools = _cache(gen, [n + p for n, p in zip(new, prefix)], kv_heads, dim, block, index, width)
    total = max(sum(new), padded)
    query, gate = (torch.randn(total, heads, dim, generator=gen).to(torch.bfloat16).to(DEV) for _ in range(2))
    cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=index, device=DEV)
    out = torch.full_like(query, 3.0)
    hip_ops.paged_attention_prefill_kv4(query, cu, torch.tensor(prefix, dtype=index, device=DEV), *pools, tables, block, max_new=max_new, gate=gate, out=out)
    untouched = torch.ones(total, dtype=torch.bool, device=DEV)
    at = 0
    for row, (n, p) in enumerate(zip(new, prefix)):
        m = min(n, max_new)
        if m:
            k, v, there = _dense(tables, pools, row, p + m, block)
            seen = (torch.arange(p + m, device=DEV)[None] <= p + torch.arange(m, device=DEV)[:, None]) & there[None]
            want, mass = _attend(query[at : at + m].double(), k, v, seen, dim**-0.5)
            _close(out[at : at + m], want, mass, gate[at : at + m])
            untouched[at : at + m] = False
        at += n
    assert (out[untouched] == 3).all()


@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 2, 256), (9, 1, 128), (6, 2, 128), (5, 1, 256)])
@pytest.mark.parametrize("width", [None, 2000])
@pytest.mark.parametrize("max_new", [1, 5, 33])
def test_tokens_past_max_new_are_not_written(heads, kv_heads, dim, width, max_new) -> None:
    _check(heads + max_new, [40, 3, 0, 20, 90], [5, 700, 9, 0, 130], max_new, heads, kv_heads, dim, 16, width)


@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 2, 256), (9, 1, 128)])
@pytest.mark.parametrize("new,prefix,max_new", [([16], [3000], 16), ([3, 17, 0, 9], [900, 0, 5, 2500], 17), ([3, 17, 0, 9], [900, 0, 5, 2500], 6)])
def test_a_step_in_a_padded_query(heads, kv_heads, dim, new, prefix, max_new) -> None:
    """The keys are split; the partial results lie by row and not by the query's row."""
    _check(heads + max_new, new, prefix, max_new, heads, kv_heads, dim, 16, 2000, padded=4096, index=torch.int64)
