"""Rows that the 4-bit operators cannot read in aligned pieces are copied to where they can, whatever makes them so."""

from __future__ import annotations

import pytest
import torch

import hip_ops


def _off_by(elements, *shape):
    """Contiguous bf16 numbers whose first one lies ``elements`` past an aligned address."""
    n = torch.Size(shape).numel()
    flat = torch.zeros(n + 8, dtype=torch.bfloat16)
    assert flat.data_ptr() % 16 == 0
    view = flat[elements : elements + n].view(shape)
    return view.copy_(torch.arange(n).remainder(251).view(shape))


def _readable(tensor, stride_t, stride_h, multiple):
    bytes_ = multiple * tensor.element_size()
    return tensor.stride(-1) == 1 and stride_t % multiple == 0 and stride_h % multiple == 0 and tensor.data_ptr() % bytes_ == 0


@pytest.mark.parametrize("shape", [(2, 8, 256), (1, 8, 128), (3, 4, 1, 256)])
@pytest.mark.parametrize("off", [1, 2, 4, 7])
@pytest.mark.parametrize("multiple", [8, 4])
def test_contiguous_rows_off_their_alignment_are_copied(shape, off, multiple) -> None:
    rows = _off_by(off, *shape)
    got, stride_t, stride_h = hip_ops._rows(rows, multiple)
    assert torch.equal(got, rows) and (stride_t, stride_h) == got.stride()[:2] and _readable(got, stride_t, stride_h, multiple)


@pytest.mark.parametrize("shape", [(1, 8, 256), (1, 8, 1, 256)])
def test_one_row_of_an_odd_stride_is_copied(shape) -> None:
    rows = torch.zeros(1, 2048 + 3, dtype=torch.bfloat16)[:, :2048].view(shape)
    rows = rows.as_strided(shape, (2051, *rows.stride()[1:]))
    got, stride_t, stride_h = hip_ops._rows(rows, 8)
    assert torch.equal(got, rows) and _readable(got, stride_t, stride_h, 8)


def test_aligned_rows_stay_where_they_are() -> None:
    proj = torch.zeros(3, 4, 512, dtype=torch.bfloat16)
    got, stride_t, stride_h = hip_ops._rows(proj[..., 256:], 8)
    assert got.data_ptr() == proj.data_ptr() + 512 and (stride_t, stride_h) == (2048, 512)


def test_the_gate_off_its_alignment_is_copied() -> None:
    gate = _off_by(1, 2, 8 * 128)
    got, at, stride_t, stride_h = hip_ops._kv4_gate(gate, 2, 8, 128, gate.device)
    assert torch.equal(got.view(2, -1), gate) and at == got.data_ptr() and _readable(got, stride_t, stride_h, 4)
