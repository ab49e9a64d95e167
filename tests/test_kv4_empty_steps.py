"""Calls with no token, no row or nothing to read do nothing and are no error: empty tensors have no address."""

from __future__ import annotations

import ctypes

import pytest
import torch

import hip_loader as L
import hip_ops
from test_kv4_refusals import SOME, P, _desc, _lib

DEV = "cuda:0"


def _prefill(lib, total, max_new, batch=2, rows=P(0), out=P(0), tables=SOME) -> int:
    return lib.qa_paged_attention_prefill_kv4(rows, L.QA_BF16, 4096, 256, total, SOME, SOME, L.QA_I32, batch, max_new, 16, 256, ctypes.byref(_desc()), tables, L.QA_I32, 4, 4, 16, 0.0,
                                              P(0), 0, 0, out, P(0), 0, P(0))


def test_prefill_without_tokens_or_rows() -> None:
    lib = _lib()
    assert _prefill(lib, 0, 0) == 0 and _prefill(lib, 0, 5) == 0
    assert _prefill(lib, 4, 0, rows=SOME, out=SOME) == 0 and _prefill(lib, 4, 4, batch=0, rows=SOME, out=SOME, tables=P(0)) == 0
    assert _prefill(lib, 4, 4) == 1 and "non-null" in L.last_error(lib)


def test_gather_of_no_rows() -> None:
    lib = _lib()
    gather = lambda batch, valid: lib.qa_paged_kv4_gather(ctypes.byref(_desc()), 256, batch, P(0), L.QA_I32, 4, 4, valid, 16, P(0), P(0), P(0))  # noqa: E731
    assert gather(0, 16) == 0
    assert gather(1, 16) == 1 and "device array" in L.last_error(lib)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,sections", [(256, (11, 11, 10)), (128, (16, 24, 24))])
def test_a_layer_without_tokens(dim, sections) -> None:
    heads, kv_heads, block = 16, 2, 16
    bf = lambda *shape: torch.zeros(*shape, dtype=torch.bfloat16, device=DEV)  # noqa: E731
    pools = [torch.zeros(2, kv_heads, hip_ops.kv4_tile_bytes(dim, block), dtype=torch.uint8, device=DEV) for _ in range(2)]
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    none = torch.zeros(0, dtype=torch.int64, device=DEV)
    prologue = lambda q, k, v: hip_ops.qk_norm_mrope_kv_append(q, k, v, bf(dim), bf(dim), torch.zeros(3, 0, dtype=torch.int64, device=DEV), sections, *pools, none, block, eps=1e-6,  # noqa: E731
                                                               rope_theta=1e6)
    for query, gate in (prologue(bf(0, heads, 2 * dim), bf(0, kv_heads, dim), bf(0, kv_heads, dim)), prologue(bf(0, heads * 2 * dim), bf(0, kv_heads * dim), bf(0, kv_heads * dim))):
        assert query.shape == gate.shape == (0, heads, dim)
        hip_ops.paged_kv4_append(bf(0, kv_heads, dim), bf(0, kv_heads, dim), *pools, none, block)
        out = hip_ops.paged_attention_prefill_kv4(query, i32(0, 0, 0), i32(0, 7), *pools, torch.zeros(2, 3, dtype=torch.int32, device=DEV), block, max_new=0, gate=gate)
        assert out.shape == (0, heads, dim)
        assert hip_ops.paged_attention_decode_kv4(query.unsqueeze(2), torch.zeros(0, 3, dtype=torch.int32, device=DEV), *pools, none, block).shape == (0, heads, 1, dim)
    tables = torch.zeros(2, 3, dtype=torch.int32, device=DEV)
    assert hip_ops.paged_kv4_gather(*pools, tables[:0], 16, block)[0].shape == (0, kv_heads, 16, dim)
    assert hip_ops.paged_kv4_gather(*pools, tables, 0, block)[0].shape == (2, kv_heads, 0, dim)
    assert not pools[0].any() and not pools[1].any()
