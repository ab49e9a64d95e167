"""Python operator surface of the gfx950 hot path.

The names, arguments, return shapes and ``RuntimeError`` behaviour of the three
hot wrappers of the reference's ``src/fp8_cuda.py`` are kept:

* :func:`paged_attention_decode` -- ``src/fp8_cuda.py:217-232``
* :func:`paged_attention_decode_batched` -- ``src/fp8_cuda.py:235-250``
* :func:`linear_attention_recurrent_core` -- ``src/fp8_cuda.py:206-214``

so a caller such as ``src/tp_runtime.py:613-643`` / ``:2778-2787`` only changes
its import.  Beyond the reference they also accept bfloat16 tensors, a shared
GQA-native block pool ``(P, H_kv, bs, D)`` and int32 tables.  New operators of
the path sit beside them (KV append/gather, prefill, conv1d, chunked delta
rule, fused decode step).

Every operator validates on the host and raises ``RuntimeError`` with the
library's message on failure.  Outputs and workspaces are allocated here with
torch (its caching allocator owns them); kernels run on torch's current stream.
"""

from __future__ import annotations

import ctypes
import math
from array import array
from typing import Any, NamedTuple, Sequence

import torch

import hip_loader as L

_DTYPE_CODES = {
    torch.float32: L.QA_F32,
    torch.bfloat16: L.QA_BF16,
    torch.float16: L.QA_F16,
    torch.int32: L.QA_I32,
    torch.int64: L.QA_I64,
}


_FLOAT_DTYPES = (torch.float32, torch.bfloat16)
_INDEX_DTYPES = (torch.int32, torch.int64)


def _code(tensor: torch.Tensor) -> int:
    try:
        return _DTYPE_CODES[tensor.dtype]
    except KeyError as exc:
        raise RuntimeError(f"unsupported dtype {tensor.dtype}") from exc


# The smallest calls are bound by this file and not by their kernels, so what every call runs stays lean: the
# raw stream handle without a Stream object, pointers as plain integers, no message formatted before a check fails.
def _stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


def _ptr(tensor: torch.Tensor | None) -> int:
    return 0 if tensor is None else tensor.data_ptr()


def _flat(tensor: torch.Tensor) -> torch.Tensor:
    return tensor if tensor.dim() == 1 else tensor.reshape(-1)


def _vector_on(tensor: torch.Tensor, device: torch.device) -> torch.Tensor:
    flat = _flat(tensor)
    return (flat if flat.device == device else flat.to(device=device)).contiguous()


def _require(cond: bool, message: str) -> None:
    if not cond:
        raise RuntimeError(message)


def _require_cuda(tensor: Any, name: str, device: torch.device | None = None) -> None:
    if not (isinstance(tensor, torch.Tensor) and tensor.is_cuda):
        raise RuntimeError(f"{name} must be CUDA")
    if device is not None and tensor.device != device:
        raise RuntimeError(f"{name} must be on same CUDA device as query")


def _float_dtype(tensor: torch.Tensor, name: str) -> None:
    if tensor.dtype not in _FLOAT_DTYPES:
        raise RuntimeError(f"{name} must be float32 or bfloat16")


def _index_dtype(tensor: torch.Tensor, name: str) -> None:
    if tensor.dtype not in _INDEX_DTYPES:
        raise RuntimeError(f"{name} must be int64/torch.long or int32")


def _pool_descriptor(key_pool: torch.Tensor, value_pool: torch.Tensor, layout: str) -> L.PagedKV:
    """Descriptor for a reference-layout ``(B, heads, P, bs, D)`` pool or a shared ``(P, H_kv, bs, D)`` pool."""
    _require(key_pool.shape == value_pool.shape, "key/value physical block count must match")
    _require(key_pool.dtype == value_pool.dtype, "key/value blocks must have the same dtype")
    _require(key_pool.stride(-1) == 1 and value_pool.stride(-1) == 1, "key/value blocks must be contiguous in head_dim")
    _require(key_pool.stride() == value_pool.stride(), "key/value blocks must share strides")
    shape, strides = key_pool.shape, key_pool.stride()
    if layout == "reference":  # (B, heads, P, bs, D)
        heads, blocks = shape[1], shape[2]
        stride_batch, stride_head, stride_block, stride_token = strides[:4]
    else:  # shared (P, H_kv, bs, D)
        blocks, heads = shape[0], shape[1]
        stride_batch = 0
        stride_block, stride_head, stride_token = strides[:3]
    return L.PagedKV(key_pool.data_ptr(), value_pool.data_ptr(), None, None, None, blocks, stride_batch, stride_block, stride_head,
                     stride_token, heads, _code(key_pool))


def _decode_workspace(lib: Any, batch: int, heads: int, head_dim: int, max_tokens: int, block_size: int, device: torch.device) -> torch.Tensor:
    nbytes = int(lib.qa_paged_attention_decode_workspace(batch, heads, head_dim, max_tokens, block_size))
    return torch.empty(max(nbytes, 4), dtype=torch.uint8, device=device)


def paged_attention_decode(
    query: torch.Tensor,
    block_table: torch.Tensor,
    key_blocks: torch.Tensor,
    value_blocks: torch.Tensor,
    sequence_length: int,
    block_size: int,
    *,
    scale: float | None = None,
) -> torch.Tensor:
    """Single-token paged attention over one block table.

    ``query`` ``(B, H, 1, D)``; ``block_table`` ``(L,)``; ``key_blocks`` either
    the reference's per-request pool ``(B, heads, P, bs, D)`` with ``heads`` = H
    or H_kv (GQA), or a shared pool ``(P, H_kv, bs, D)``.  Returns
    ``(B, H, 1, D)`` in the query dtype.  Reference:
    ``src/fp8_cuda.py:217-232`` -> ``src/csrc/fp8_linear_cuda.cu:1192-1266``.
    """
    lib = L.load_library()
    _require_cuda(query, "query")
    device = query.device
    _require_cuda(block_table, "block_table", device)
    _require_cuda(key_blocks, "key_blocks", device)
    _require_cuda(value_blocks, "value_blocks", device)
    _float_dtype(query, "query")
    _float_dtype(key_blocks, "key_blocks")
    _index_dtype(block_table, "block_table")
    _require(query.dim() == 4, "query must have shape [batch, heads, 1, head_dim]")
    _require(query.shape[2] == 1, "query seq_len must be 1 for paged decode")
    _require(block_table.dim() == 1, "block_table must be rank-1")
    _require(key_blocks.dim() in (4, 5), "key_blocks must have shape [batch, heads, blocks, block_size, head_dim] or [blocks, kv_heads, block_size, head_dim]")
    _require(value_blocks.dim() == key_blocks.dim(), "value_blocks must match key_blocks rank")
    _require(int(sequence_length) > 0, "sequence_length must be positive")
    _require(int(block_size) > 0, "block_size must be positive")
    batch, heads, _, head_dim = query.shape
    layout = "reference" if key_blocks.dim() == 5 else "shared"
    if layout == "reference":
        _require(key_blocks.shape[0] == batch and value_blocks.shape[0] == batch, "KV batch must match query")
    _require(key_blocks.shape[-2] == block_size, "KV block_size mismatch")
    _require(key_blocks.shape[-1] == head_dim, "KV head_dim must match query")
    table = block_table.contiguous()
    _require(table.numel() * int(block_size) >= int(sequence_length), "block_table does not cover sequence_length")
    q = query.contiguous()
    desc = _pool_descriptor(key_blocks, value_blocks, layout)
    _require(heads % desc.kv_heads == 0, "KV heads must divide query heads")
    out = torch.empty_like(q)
    ws = _decode_workspace(lib, batch, heads, head_dim, int(sequence_length), int(block_size), device)
    status = lib.qa_paged_attention_decode(
        _ptr(q), _code(q), q.stride(0), q.stride(1), batch, heads, head_dim, ctypes.byref(desc), _ptr(table), _code(table),
        table.numel(), int(sequence_length), int(block_size), float(scale or 0.0), _ptr(out), _ptr(ws), ws.numel(), _stream(device),
    )
    L.check(lib, status, "paged_attention_decode")
    return out


def paged_attention_decode_batched(
    query: torch.Tensor,
    block_tables: torch.Tensor,
    key_blocks: Sequence[torch.Tensor] | torch.Tensor,
    value_blocks: Sequence[torch.Tensor] | torch.Tensor,
    sequence_lengths: torch.Tensor,
    block_size: int,
    *,
    scale: float | None = None,
) -> torch.Tensor:
    """Batched single-token paged attention with per-row tables and lengths.

    ``block_tables`` ``(B, max_blocks)`` padded with -1, ``sequence_lengths``
    ``(B,)``.  ``key_blocks``/``value_blocks`` are either one shared
    ``(P, H_kv, bs, D)`` pool, or (as the reference) a list of per-request
    pools ``(1, heads, P_b, bs, D)``; a list whose entries are all the same
    tensor is treated as one shared pool.  Rows of length <= 0 give zeros.
    Reference: ``src/fp8_cuda.py:235-250`` -> ``src/csrc/fp8_linear_cuda.cu:1269-1365``.
    """
    lib = L.load_library()
    _require_cuda(query, "query")
    device = query.device
    _require_cuda(block_tables, "block_tables", device)
    _require_cuda(sequence_lengths, "sequence_lengths", device)
    _float_dtype(query, "query")
    _index_dtype(block_tables, "block_tables")
    _index_dtype(sequence_lengths, "sequence_lengths")
    _require(query.dim() == 4, "query must have shape [batch, heads, 1, head_dim]")
    _require(block_tables.dim() == 2, "block_tables must have shape [batch, max_blocks]")
    _require(sequence_lengths.dim() == 1, "sequence_lengths must be rank-1")
    _require(query.shape[2] == 1, "query seq_len must be 1 for paged decode")
    _require(int(block_size) > 0, "block_size must be positive")
    batch, heads, _, head_dim = query.shape
    _require(block_tables.shape[0] == batch, "block_tables batch must match query")
    _require(sequence_lengths.shape[0] == batch, "sequence_lengths batch must match query")
    _require(block_tables.shape[1] > 0, "max_blocks must be positive and fit int32")
    keepalive: list[torch.Tensor] = []
    if isinstance(key_blocks, torch.Tensor):
        _require(isinstance(value_blocks, torch.Tensor), "value_blocks must match key_blocks")
        _require(key_blocks.dim() == 4, "shared pools must have shape [blocks, kv_heads, block_size, head_dim]")
        _require_cuda(key_blocks, "key_blocks", device)
        _require_cuda(value_blocks, "value_blocks", device)
        _float_dtype(key_blocks, "key_blocks")
        desc = _pool_descriptor(key_blocks, value_blocks, "shared")
        pool_block_size = key_blocks.shape[2]
    else:
        key_list = list(key_blocks)
        value_list = list(value_blocks)
        _require(len(key_list) == batch, "key_blocks list length must match batch")
        _require(len(value_list) == batch, "value_blocks list length must match batch")
        first_k, first_v = key_list[0], value_list[0]
        for k, v in zip(key_list, value_list):
            _require(isinstance(k, torch.Tensor) and isinstance(v, torch.Tensor), "key/value blocks must be CUDA")
            _require(k.is_cuda and v.is_cuda, "key/value blocks must be CUDA")
            _require(k.device == device and v.device == device, "key/value blocks must be on same CUDA device as query")
            _require(k.dtype == first_k.dtype and v.dtype == first_k.dtype, "key/value blocks must share one dtype")
            _float_dtype(k, "key/value blocks")
            _require(k.dim() == first_k.dim() and v.dim() == first_k.dim(), "key/value blocks must share one rank")
            _require(k.shape == v.shape, "key/value physical block count must match")
        shared = all(k is first_k for k in key_list) and all(v is first_v for v in value_list)
        if shared and first_k.dim() == 4:
            desc = _pool_descriptor(first_k, first_v, "shared")
            pool_block_size = first_k.shape[2]
        else:
            for k in key_list:
                _require(k.dim() == 5, "key/value blocks must have shape [1, heads, blocks, block_size, head_dim]")
                _require(k.shape[0] == 1, "per-request KV pools must have batch dim 1")
                _require(k.shape[1] == first_k.shape[1], "KV heads must match across pools")
                _require(k.shape[3:] == first_k.shape[3:], "KV block_size/head_dim must match across pools")
                _require(k.stride(-1) == 1 and k.is_contiguous(), "key/value blocks must be contiguous")
            for v in value_list:
                _require(v.is_contiguous(), "key/value blocks must be contiguous")
            desc = _per_request_descriptor(key_list, value_list, device, keepalive)
            pool_block_size = first_k.shape[3]
    _require(pool_block_size == block_size, "KV block_size mismatch")
    _require(heads % desc.kv_heads == 0, "KV heads must divide query heads")
    q = query.contiguous()
    tables = block_tables.contiguous()
    lens = sequence_lengths.contiguous()
    max_blocks = tables.shape[1]
    out = torch.empty_like(q)
    ws = _decode_workspace(lib, batch, heads, head_dim, max_blocks * int(block_size), int(block_size), device)
    status = lib.qa_paged_attention_decode_batched(
        _ptr(q), _code(q), q.stride(0), q.stride(1), batch, heads, head_dim, ctypes.byref(desc), _ptr(tables), _code(tables),
        tables.stride(0), max_blocks, _ptr(lens), _code(lens), int(block_size), float(scale or 0.0), _ptr(out), _ptr(ws), ws.numel(),
        _stream(device),
    )
    L.check(lib, status, "paged_attention_decode_batched")
    return out


def paged_attention_decode_batched_noalloc(
    query: torch.Tensor,
    block_tables: torch.Tensor,
    key_blocks: torch.Tensor,
    value_blocks: torch.Tensor,
    sequence_lengths: torch.Tensor,
    block_size: int,
    *,
    scale: float | None = None,
) -> torch.Tensor:
    """``paged_attention_decode_batched`` on one shared ``(P, H_kv, bs, D)`` pool with the split-K
    partials in the library's static per-device scratch (``qa_paged_attention_decode_batched_noalloc``):
    the library allocates nothing; only the output is a new tensor.  Sizes whose partials exceed the
    scratch raise ``RuntimeError``; calls that overlap on one device race."""
    lib = L.load_library()
    _require_cuda(query, "query")
    device = query.device
    for tensor, name in ((block_tables, "block_tables"), (sequence_lengths, "sequence_lengths"), (key_blocks, "key_blocks"),
                         (value_blocks, "value_blocks")):
        _require_cuda(tensor, name, device)
    _float_dtype(query, "query")
    _float_dtype(key_blocks, "key_blocks")
    _index_dtype(block_tables, "block_tables")
    _index_dtype(sequence_lengths, "sequence_lengths")
    _require(query.dim() == 4 and query.shape[2] == 1, "query must have shape [batch, heads, 1, head_dim]")
    _require(key_blocks.dim() == 4 and value_blocks.shape == key_blocks.shape, "shared pools must have shape [blocks, kv_heads, block_size, head_dim]")
    batch, heads, _, head_dim = query.shape
    _require(block_tables.dim() == 2 and block_tables.shape[0] == batch and block_tables.shape[1] > 0, "block_tables must have shape [batch, max_blocks]")
    _require(sequence_lengths.dim() == 1 and sequence_lengths.shape[0] == batch, "sequence_lengths batch must match query")
    _require(key_blocks.shape[2] == block_size, "KV block_size mismatch")
    desc = _pool_descriptor(key_blocks, value_blocks, "shared")
    _require(heads % desc.kv_heads == 0, "KV heads must divide query heads")
    q = query.contiguous()
    tables = block_tables.contiguous()
    lens = sequence_lengths.contiguous()
    out = torch.empty_like(q)
    status = lib.qa_paged_attention_decode_batched_noalloc(
        _ptr(q), _code(q), q.stride(0), q.stride(1), batch, heads, head_dim, ctypes.byref(desc), _ptr(tables), _code(tables),
        tables.stride(0), tables.shape[1], _ptr(lens), _code(lens), int(block_size), float(scale or 0.0), _ptr(out), _stream(device),
    )
    L.check(lib, status, "paged_attention_decode_batched_noalloc")
    return out


def _per_request_descriptor(key_list: list[torch.Tensor], value_list: list[torch.Tensor], device: torch.device, keepalive: list[torch.Tensor]) -> L.PagedKV:
    """Pointer-array descriptor for contiguous per-request pools ``(1, heads, P_b, bs, D)``.

    As the reference host wrapper (``src/csrc/fp8_linear_cuda.cu:1308-1340``),
    row pointers and block counts are copied to the device for each call.
    ``stride_head = 0`` tells the kernels that row ``b``'s head stride is
    ``P_b * stride_block`` (pools of different ``P_b``).
    """
    first = key_list[0]
    key_ptrs = torch.tensor([k.data_ptr() for k in key_list], dtype=torch.int64, device=device)
    value_ptrs = torch.tensor([v.data_ptr() for v in value_list], dtype=torch.int64, device=device)
    counts = torch.tensor([k.shape[2] for k in key_list], dtype=torch.int64, device=device)
    keepalive.extend([key_ptrs, value_ptrs, counts])
    desc = L.PagedKV()
    desc.key = None
    desc.value = None
    desc.row_key_ptrs = key_ptrs.data_ptr()
    desc.row_value_ptrs = value_ptrs.data_ptr()
    desc.row_blocks = counts.data_ptr()
    desc.num_blocks = max(k.shape[2] for k in key_list)
    desc.stride_batch = 0
    desc.stride_head = 0
    desc.stride_block = first.stride(2)
    desc.stride_token = first.stride(3)
    desc.kv_heads = first.shape[1]
    desc.dtype = _code(first)
    return desc


def paged_kv_append(
    key: torch.Tensor,
    value: torch.Tensor,
    key_pool: torch.Tensor,
    value_pool: torch.Tensor,
    block_tables: torch.Tensor,
    starts: torch.Tensor | int,
    block_size: int,
    *,
    counts: torch.Tensor | None = None,
) -> None:
    """Write new K/V ``(B, H_kv, S, D)`` into pool slots in place (bit-exact).

    Row ``b`` token ``s`` goes to slot ``(table[b][(start_b+s)//bs], (start_b+s)%bs)``
    of the shared pool ``(P, H_kv, bs, D)`` or of the reference-layout pool
    ``(B, heads, P, bs, D)``.  ``block_tables`` is ``(B, max_blocks)`` or a single
    ``(max_blocks,)`` table shared by all rows.  Replaces the fragment loop of
    ``FullAttentionCache.append_blocks`` (``src/decode_state.py:271-293``).
    """
    lib = L.load_library()
    _require_cuda(key, "key")
    device = key.device
    for tensor, name in ((value, "value"), (key_pool, "key_pool"), (value_pool, "value_pool"), (block_tables, "block_tables")):
        _require_cuda(tensor, name, device)
    _require(key.shape == value.shape and key.dim() == 4, "key/value must have shape [batch, kv_heads, seq, head_dim]")
    _require(key.dtype == key_pool.dtype and value.dtype == key_pool.dtype, "new KV dtype must match the pool dtype")
    _require(key.stride() == value.stride() and key.stride(-1) == 1, "key/value must share strides with a contiguous head_dim")
    _index_dtype(block_tables, "block_tables")
    layout = "reference" if key_pool.dim() == 5 else "shared"
    desc = _pool_descriptor(key_pool, value_pool, layout)
    batch, kv_heads, seq, head_dim = key.shape
    _require(kv_heads == desc.kv_heads, "new KV heads must match the pool")
    _require(key_pool.shape[-1] == head_dim and key_pool.shape[-2] == block_size, "pool block_size/head_dim mismatch")
    tables = block_tables.contiguous()
    table_stride = tables.stride(0) if tables.dim() == 2 else 0
    max_blocks = tables.shape[-1]
    start_ptr, start_code, start_scalar = 0, L.QA_I64, 0
    if isinstance(starts, torch.Tensor):
        _require_cuda(starts, "starts", device)
        _index_dtype(starts, "starts")
        starts = starts.contiguous()
        start_ptr, start_code = _ptr(starts), _code(starts)
    else:
        start_scalar = int(starts)
    count_ptr, count_code = 0, L.QA_I64
    if counts is not None:
        _require_cuda(counts, "counts", device)
        _index_dtype(counts, "counts")
        counts = counts.contiguous()
        count_ptr, count_code = _ptr(counts), _code(counts)
    status = lib.qa_paged_kv_append(
        _ptr(key), _ptr(value), _code(key), key.stride(0), key.stride(1), key.stride(2), batch, kv_heads, seq, head_dim,
        ctypes.byref(desc), _ptr(tables), _code(tables), table_stride, max_blocks, start_ptr, start_code, start_scalar,
        count_ptr, count_code, int(block_size), _stream(device),
    )
    L.check(lib, status, "paged_kv_append")


def paged_kv_reserve(
    block_tables: torch.Tensor,
    lengths: torch.Tensor,
    free_list: torch.Tensor,
    free_state: torch.Tensor,
    status: torch.Tensor,
    block_size: int,
    *,
    counts: torch.Tensor | int = 1,
    positions: torch.Tensor | None = None,
) -> None:
    """Reserve the blocks a batched step needs, on the device (no host round trip).

    Row ``b`` grows from ``lengths[b]`` to ``lengths[b] + counts_b`` tokens: its new
    logical blocks get ids from the head of the ascending ``free_list`` (int32),
    rows in order -- the reference's lowest-free-id policy
    (``src/decode_state.py:72-78``).  ``free_state`` (int32 ``[head, count]``) is
    advanced, ``lengths`` are advanced in place, ``positions`` (if given) receives
    the old lengths.  ``status`` (int32 ``[1]``) becomes 0, or 1 (pool exhausted),
    2 (a table row too short), 3 (corrupt free state), 4 (negative or overflowing
    length or count), in which case nothing else is written.  Every argument is a
    device tensor and nothing is read back, so the call can be captured in a HIP graph.
    """
    lib = L.load_library()
    _require_cuda(block_tables, "block_tables")
    device = block_tables.device
    for tensor, name in ((lengths, "lengths"), (free_list, "free_list"), (free_state, "free_state"), (status, "status")):
        _require_cuda(tensor, name, device)
    _index_dtype(block_tables, "block_tables")
    _index_dtype(lengths, "lengths")
    _require(block_tables.dim() == 2 and block_tables.stride(1) == 1, "block_tables must have shape [batch, max_blocks] with contiguous rows")
    _require(lengths.dim() == 1 and lengths.is_contiguous() and lengths.shape[0] == block_tables.shape[0], "lengths must be a contiguous [batch] tensor")
    _require(free_list.dtype == torch.int32 and free_list.dim() == 1 and free_list.is_contiguous(), "free_list must be a contiguous int32 vector")
    _require(free_state.dtype == torch.int32 and free_state.numel() == 2 and free_state.is_contiguous(), "free_state must be int32 [head, count]")
    _require(status.dtype == torch.int32 and status.numel() >= 1, "status must be an int32 tensor")
    count_ptr, count_code, count_scalar = 0, L.QA_I64, 0
    if isinstance(counts, torch.Tensor):
        _require_cuda(counts, "counts", device)
        _index_dtype(counts, "counts")
        _require(counts.dim() == 1 and counts.is_contiguous() and counts.shape[0] == lengths.shape[0], "counts must be a contiguous [batch] tensor")
        count_ptr, count_code = _ptr(counts), _code(counts)
    else:
        count_scalar = int(counts)
        _require(count_scalar >= 0, "counts must be non-negative")
    pos_ptr, pos_code = 0, L.QA_I64
    if positions is not None:
        _require_cuda(positions, "positions", device)
        _index_dtype(positions, "positions")
        _require(positions.dim() == 1 and positions.is_contiguous() and positions.shape[0] == lengths.shape[0], "positions must be a contiguous [batch] tensor")
        pos_ptr, pos_code = _ptr(positions), _code(positions)
    status_code = lib.qa_paged_kv_reserve(
        _ptr(block_tables), _code(block_tables), block_tables.stride(0), block_tables.shape[1], _ptr(lengths), _code(lengths),
        pos_ptr, pos_code, count_ptr, count_code, count_scalar, lengths.shape[0], int(block_size), _ptr(free_list),
        free_list.numel(), _ptr(free_state), _ptr(status), _stream(device),
    )
    L.check(lib, status_code, "paged_kv_reserve")


class PackedFp8Weight:
    """An fp8 E4M3 weight re-laid by ``fp8_pack_weight`` (same bytes, streaming order)."""

    def __init__(self, data: torch.Tensor, out_features: int, in_features: int) -> None:
        self.data = data
        self.shape = (out_features, in_features)
        self.device = data.device


def fp8_pack_weight(weight: torch.Tensor) -> PackedFp8Weight:
    """Re-lay an ``(N, K)`` fp8 weight once (at load time) into 16 x 128 tiles of 2 KB, consecutive
    along K, in the order the linear kernel reads them: each wave then streams contiguous memory.
    No counterpart in the reference, whose weights stay row-major."""
    lib = L.load_library()
    _require_cuda(weight, "weight")
    _require(weight.dtype in (torch.float8_e4m3fn, torch.uint8) and weight.dim() == 2, "weight must be a rank-2 torch.float8_e4m3fn tensor")
    rows, cols = weight.shape
    _require(rows % 128 == 0 and cols % 128 == 0, "weight rows and cols must be divisible by 128 for the FP8 op")
    src = weight.contiguous()
    dst = torch.empty((rows * cols,), dtype=torch.uint8, device=weight.device)
    L.check(lib, lib.qa_fp8_pack_weight(_ptr(src), _ptr(dst), rows, cols, _stream(weight.device)), "fp8_pack_weight")
    return PackedFp8Weight(dst, rows, cols)


def fp8_e4m3_bf16_linear(input: torch.Tensor, weight: torch.Tensor | PackedFp8Weight, scale: torch.Tensor, *, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """``y = input @ (E4M3(weight) * block scale)^T`` with 128 x 128 bf16 scale blocks.

    Same name, arguments and result as the reference's ``fp8_cuda.fp8_e4m3_bf16_linear``
    (``src/fp8_cuda.py:16-17`` -> ``src/csrc/fp8_linear_cuda.cu:1368-1466``): ``weight``
    ``(N, K)`` ``torch.float8_e4m3fn`` (or its uint8 codes), ``scale`` ``(N/128, K/128)``
    bf16, ``input`` ``(..., K)`` float32 (bf16 also accepted); returns ``(..., N)`` float32
    (or ``out_dtype`` bf16).  N and K must be multiples of 128, as in the reference's op.
    ``weight`` may also be the ``fp8_pack_weight`` form of the same weight (faster streaming).
    """
    lib = L.load_library()
    _require_cuda(input, "input")
    device = input.device
    _require_cuda(weight.data if isinstance(weight, PackedFp8Weight) else weight, "weight", device)
    _require_cuda(scale, "scale", device)
    _require(input.dtype in (torch.float32, torch.bfloat16), "input must be float32 or bfloat16")
    packed = isinstance(weight, PackedFp8Weight)
    _require(packed or weight.dtype in (torch.float8_e4m3fn, torch.uint8), "weight must be torch.float8_e4m3fn")
    _require(scale.dtype == torch.bfloat16, "scale must be bfloat16")
    _require(packed or weight.dim() == 2, "weight must be rank-2")
    _require(scale.dim() == 2, "scale must be rank-2")
    _require(input.dim() >= 2, "input must be at least rank-2")
    _require(out_dtype in (torch.float32, torch.bfloat16), "out_dtype must be float32 or bfloat16")
    rows, cols = weight.shape
    _require(input.shape[-1] == cols, "input last dim must match weight cols")
    _require(rows % 128 == 0, "weight rows must be divisible by 128 for the FP8 op")
    _require(cols % 128 == 0, "weight cols must be divisible by 128 for the FP8 op")
    _require(scale.shape == (rows // 128, cols // 128), "scale blocks mismatch")
    x = input.contiguous()
    if x.dim() != 2:
        x = x.view(-1, cols)
    w = weight.data if packed else weight.contiguous()
    s = scale.contiguous()
    out = torch.empty((x.shape[0], rows), dtype=out_dtype, device=device)
    nbytes = int(lib.qa_fp8_linear_workspace(x.shape[0], rows, cols))
    ws = torch.empty(max(nbytes, 4), dtype=torch.uint8, device=device)
    status = lib.qa_fp8_linear(
        _ptr(x), _code(x), x.stride(0), x.shape[0], _ptr(w), int(packed), _ptr(s), rows, cols, _ptr(out), _code(out), out.stride(0), _ptr(ws),
        ws.numel(), _stream(device),
    )
    L.check(lib, status, "fp8_e4m3_bf16_linear")
    return out if input.dim() == 2 else out.view(*input.shape[:-1], rows)


def paged_kv_gather(key_pool: torch.Tensor, value_pool: torch.Tensor, block_tables: torch.Tensor, valid: int, block_size: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Dense ``(B, H_kv, valid, D)`` logical-order K/V (``src/decode_state.py:295-303,395-404``)."""
    lib = L.load_library()
    _require_cuda(key_pool, "key_pool")
    device = key_pool.device
    _require_cuda(value_pool, "value_pool", device)
    _require_cuda(block_tables, "block_tables", device)
    _index_dtype(block_tables, "block_tables")
    layout = "reference" if key_pool.dim() == 5 else "shared"
    desc = _pool_descriptor(key_pool, value_pool, layout)
    tables = block_tables.contiguous()
    if tables.dim() == 1:
        tables = tables.unsqueeze(0)
    batch = tables.shape[0] if layout == "shared" else key_pool.shape[0]
    table_stride = tables.stride(0) if tables.shape[0] > 1 else 0
    head_dim = key_pool.shape[-1]
    key_out = torch.empty((batch, desc.kv_heads, int(valid), head_dim), dtype=key_pool.dtype, device=device)
    value_out = torch.empty_like(key_out)
    status = lib.qa_paged_kv_gather(
        ctypes.byref(desc), head_dim, batch, _ptr(tables), _code(tables), table_stride, tables.shape[1], int(valid), int(block_size),
        _ptr(key_out), _ptr(value_out), _stream(device),
    )
    L.check(lib, status, "paged_kv_gather")
    return key_out, value_out


# --------------------------------------------------------------------------- gated delta rule


def _f32_contig(tensor: torch.Tensor, name: str, device: torch.device) -> torch.Tensor:
    _require_cuda(tensor, name, device)
    _require(tensor.dtype == torch.float32, f"{name} must be float32")
    return tensor.contiguous()


def linear_attention_recurrent_core(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, g: torch.Tensor, beta: torch.Tensor, initial_state: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Token-serial gated delta rule on prepared inputs.

    ``query``/``key`` ``(B, H, S, dk)``, ``value`` ``(B, H, S, dv)``,
    ``g``/``beta`` ``(B, H, S)``, ``initial_state`` ``(B, H, dk, dv)``, all
    float32 (already L2-normalised and scaled, ``src/tp_runtime.py:2790-2805``).
    Returns ``(output (B, H, S, dv), final_state)`` fp32.  Reference:
    ``src/fp8_cuda.py:206-214`` -> ``src/csrc/fp8_linear_cuda.cu:2491-2573``.
    """
    lib = L.load_library()
    _require_cuda(query, "query")
    device = query.device
    q = _f32_contig(query, "query", device)
    k = _f32_contig(key, "key", device)
    v = _f32_contig(value, "value", device)
    gg = _f32_contig(g, "g", device)
    bb = _f32_contig(beta, "beta", device)
    s0 = _f32_contig(initial_state, "initial_state", device)
    _require(q.dim() == 4, "query must have shape [batch, heads, seq_len, key_dim]")
    _require(k.dim() == 4, "key must have shape [batch, heads, seq_len, key_dim]")
    _require(v.dim() == 4, "value must have shape [batch, heads, seq_len, value_dim]")
    _require(gg.dim() == 3, "g must have shape [batch, heads, seq_len]")
    _require(bb.dim() == 3, "beta must have shape [batch, heads, seq_len]")
    _require(s0.dim() == 4, "initial_state must have shape [batch, heads, key_dim, value_dim]")
    batch, heads, seq, key_dim = q.shape
    value_dim = v.shape[3]
    _require(batch > 0 and heads > 0 and seq > 0 and key_dim > 0 and value_dim > 0, "seq_len must be positive and fit int32")
    _require(k.shape == q.shape, "key shape must match query shape")
    _require(tuple(v.shape[:3]) == (batch, heads, seq), "value batch/head/seq must match query")
    _require(tuple(gg.shape) == (batch, heads, seq), "g shape must match [batch, heads, seq_len]")
    _require(tuple(bb.shape) == (batch, heads, seq), "beta shape must match [batch, heads, seq_len]")
    _require(tuple(s0.shape[:2]) == (batch, heads), "initial_state batch/head must match query")
    _require(tuple(s0.shape[2:]) == (key_dim, value_dim), "initial_state key/value dims must match query/value")
    out = torch.empty((batch, heads, seq, value_dim), dtype=torch.float32, device=device)
    final = torch.empty_like(s0)
    status = lib.qa_linear_attention_recurrent_core(
        _ptr(q), _ptr(k), _ptr(v), _ptr(gg), _ptr(bb), _ptr(s0), _ptr(out), _ptr(final), batch, heads, seq, key_dim, value_dim, _stream(device)
    )
    L.check(lib, status, "linear_attention_recurrent_core")
    return out, final


def _conv_weight(weight: torch.Tensor, channels: int, device: torch.device) -> torch.Tensor:
    _require_cuda(weight, "conv weight", device)
    w = weight if weight.dim() == 2 else weight.reshape(weight.shape[0], weight.shape[-1])
    if w.dtype != torch.float32 or not w.is_contiguous():
        w = w.float().contiguous()
    _require(w.shape[0] == channels, "conv weight must have one row per channel")
    return w


def causal_conv1d_prefill(
    x: torch.Tensor, weight: torch.Tensor, conv_state: torch.Tensor | None = None, *, apply_silu: bool = True, out_dtype: torch.dtype = torch.float32
) -> tuple[torch.Tensor, torch.Tensor]:
    """Depthwise causal conv1d (+SiLU) over a token-major ``(B, T, C)`` input.

    ``conv_state`` ``(B, C, K-1)`` holds the previous K-1 inputs (zeros when
    None).  Returns ``(out (B, T, C), new_state (B, C, K-1))``; the math is the
    fp32 ``F.conv1d`` of ``src/reference_ops.py:245-258``.
    """
    lib = L.load_library()
    _require_cuda(x, "x")
    device = x.device
    _require(x.dim() == 3 and x.stride(-1) == 1, "x must be (batch, seq, channels) with contiguous channels")
    _float_dtype(x, "x")
    batch, seq, channels = x.shape
    w = _conv_weight(weight, channels, device)
    kernel = w.shape[1]
    state_in = None
    if conv_state is not None:
        state_in = _f32_contig(conv_state, "conv_state", device)
        _require(tuple(state_in.shape) == (batch, channels, kernel - 1), "conv_state must be (batch, channels, kernel-1)")
    new_state = torch.empty((batch, channels, kernel - 1), dtype=torch.float32, device=device)
    out = torch.empty((batch, seq, channels), dtype=out_dtype, device=device)
    status = lib.qa_causal_conv1d_prefill(
        _ptr(x), _code(x), x.stride(0), x.stride(1), _ptr(state_in), _ptr(new_state), channels * (kernel - 1), 0, L.QA_I32,
        batch, _ptr(w), batch, seq, channels, kernel, _ptr(out), _code(out), out.stride(0), out.stride(1), int(apply_silu), _stream(device),
    )
    L.check(lib, status, "causal_conv1d_prefill")
    return out, new_state


def causal_conv1d_update(x: torch.Tensor, conv_state: torch.Tensor, weight: torch.Tensor, slots: torch.Tensor | None = None, *, apply_silu: bool = True) -> torch.Tensor:
    """One token ``x`` ``(B, C)`` through the conv; ``conv_state`` ``(rows, C, K-1)`` updated in place.

    Row ``b`` uses state row ``slots[b]`` (or ``b``).  Returns fp32 ``(B, C)``.
    """
    lib = L.load_library()
    _require_cuda(x, "x")
    device = x.device
    _require(x.dim() == 2 and x.stride(-1) == 1, "x must be (batch, channels)")
    _float_dtype(x, "x")
    batch, channels = x.shape
    w = _conv_weight(weight, channels, device)
    kernel = w.shape[1]
    _require_cuda(conv_state, "conv_state", device)
    _require(conv_state.dtype == torch.float32 and conv_state.is_contiguous(), "conv_state must be contiguous float32")
    _require(tuple(conv_state.shape[1:]) == (channels, kernel - 1), "conv_state must be (rows, channels, kernel-1)")
    slot_ptr, slot_code = 0, L.QA_I32
    if slots is not None:
        _require_cuda(slots, "slots", device)
        _index_dtype(slots, "slots")
        slots = slots.contiguous()
        slot_ptr, slot_code = _ptr(slots), _code(slots)
    out = torch.empty((batch, channels), dtype=torch.float32, device=device)
    status = lib.qa_causal_conv1d_update(
        _ptr(x), _code(x), x.stride(0), _ptr(conv_state), channels * (kernel - 1), slot_ptr, slot_code, conv_state.shape[0], _ptr(w), batch,
        channels, kernel,
        _ptr(out), L.QA_F32, out.stride(0), int(apply_silu), _stream(device),
    )
    L.check(lib, status, "causal_conv1d_update")
    return out


def gated_delta_step(
    qkv: torch.Tensor,
    a: torch.Tensor,
    b: torch.Tensor,
    a_log: torch.Tensor,
    dt_bias: torch.Tensor,
    state: torch.Tensor,
    *,
    key_heads: int,
    slots: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.bfloat16,
    z: torch.Tensor | None = None,
    norm_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
) -> torch.Tensor:
    """Fused single-token recurrence of a linear-attention layer.

    ``qkv`` ``(B, 2*Hqk*dk + Hv*dv)`` fp32 is the conv+SiLU output; ``a``/``b``
    ``(B, Hv)`` the raw ``in_proj_a``/``in_proj_b`` outputs; ``state``
    ``(slots, Hv, dk, dv)`` fp32 is updated in place at ``slots[b]`` (or ``b``).
    Returns ``(B, Hv, dv)`` in ``out_dtype``.  Follows
    ``src/reference_ops.py:271-283,291-322`` for one token.  With ``z`` (the
    ``in_proj_z`` output ``(B, Hv*dv)``) and ``norm_weight`` ``(dv,)`` the same
    kernel also applies the layer's output stage, ``gated_rms_norm`` on the fp32
    core (``src/reference_ops.py:172-178,284-287``).
    """
    lib = L.load_library()
    _require_cuda(qkv, "qkv")
    device = qkv.device
    _require(qkv.dtype == torch.float32 and qkv.dim() == 2 and qkv.stride(-1) == 1, "qkv must be (batch, channels) float32")
    _require_cuda(state, "state", device)
    _require(state.dtype == torch.float32 and state.dim() == 4 and state.is_contiguous(), "state must be contiguous (slots, Hv, dk, dv) float32")
    _, value_heads, key_dim, value_dim = state.shape
    batch = qkv.shape[0]
    _require_cuda(a, "a", device)
    _require_cuda(b, "b", device)
    _require(a.shape == (batch, value_heads) and b.shape == (batch, value_heads), "a/b must be (batch, value_heads)")
    _require(a.dtype == b.dtype and a.dtype in (torch.float32, torch.bfloat16), "a/b must share a float32/bfloat16 dtype")
    a_c, b_c = a.contiguous(), b.contiguous()
    alog = _f32_contig(_flat(a_log), "a_log", device)
    dtb = _f32_contig(_flat(dt_bias), "dt_bias", device)
    slot_ptr, slot_code = 0, L.QA_I32
    if slots is not None:
        _require_cuda(slots, "slots", device)
        _index_dtype(slots, "slots")
        slots = slots.contiguous()
        slot_ptr, slot_code = _ptr(slots), _code(slots)
    out = torch.empty((batch, value_heads, value_dim), dtype=out_dtype, device=device)
    if z is None:
        _require(norm_weight is None, "norm_weight needs z")
        status = lib.qa_gated_delta_step(
            _ptr(qkv), qkv.stride(0), _ptr(a_c), _ptr(b_c), _code(a_c), a_c.stride(0), _ptr(alog), _ptr(dtb), _ptr(state), state.stride(0),
            slot_ptr, slot_code, state.shape[0], _ptr(out), _code(out), out.stride(0), batch, int(key_heads), value_heads, key_dim, value_dim, _stream(device),
        )
    else:
        _require_cuda(z, "z", device)
        _float_dtype(z, "z")
        _require(norm_weight is not None, "the output stage needs norm_weight")
        zz = z if z.shape == (batch, value_heads * value_dim) else z.reshape(batch, value_heads * value_dim)
        _require(zz.stride(-1) == 1, "z rows must be contiguous")
        w = _vector_on(norm_weight, device)
        _float_dtype(w, "norm_weight")
        _require(w.numel() == value_dim, "norm_weight must have value_dim elements")
        status = lib.qa_gated_delta_step_norm(
            _ptr(qkv), qkv.stride(0), _ptr(a_c), _ptr(b_c), _code(a_c), a_c.stride(0), _ptr(alog), _ptr(dtb), _ptr(state), state.stride(0),
            slot_ptr, slot_code, state.shape[0], _ptr(zz), _code(zz), zz.stride(0), _ptr(w), _code(w), float(eps), _ptr(out), _code(out), out.stride(0), batch,
            int(key_heads), value_heads, key_dim, value_dim, _stream(device),
        )
    L.check(lib, status, "gated_delta_step")
    return out


def gated_delta_step_conv(
    x: torch.Tensor,
    conv_state: torch.Tensor,
    conv_weight: torch.Tensor,
    a: torch.Tensor,
    b: torch.Tensor,
    a_log: torch.Tensor,
    dt_bias: torch.Tensor,
    state: torch.Tensor,
    *,
    key_heads: int,
    slots: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.bfloat16,
    z: torch.Tensor | None = None,
    norm_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
) -> torch.Tensor:
    """``causal_conv1d_update`` followed by ``gated_delta_step`` in one kernel.

    ``x`` ``(B, C)`` is the token's raw ``in_proj_qkv`` row (float32 or bfloat16),
    ``conv_state`` ``(rows, C, K-1)`` fp32 and ``state`` ``(rows, Hv, dk, dv)`` fp32 are
    both updated in place at row ``slots[b]`` (or ``b``); the other arguments and the
    result are ``gated_delta_step``'s.  The activations and outputs equal those of the
    two calls.
    """
    lib = L.load_library()
    _require_cuda(x, "x")
    device = x.device
    _require(x.dim() == 2 and x.stride(-1) == 1, "x must be (batch, channels)")
    _float_dtype(x, "x")
    batch, channels = x.shape
    w = _conv_weight(conv_weight, channels, device)
    kernel = w.shape[1]
    _require_cuda(conv_state, "conv_state", device)
    _require(conv_state.dtype == torch.float32 and conv_state.is_contiguous(), "conv_state must be contiguous float32")
    _require(tuple(conv_state.shape[1:]) == (channels, kernel - 1), "conv_state must be (rows, channels, kernel-1)")
    _require_cuda(state, "state", device)
    _require(state.dtype == torch.float32 and state.dim() == 4 and state.is_contiguous(), "state must be contiguous (slots, Hv, dk, dv) float32")
    _require(conv_state.shape[0] == state.shape[0], "conv_state and state must have the same rows")
    _, value_heads, key_dim, value_dim = state.shape
    _require(channels == 2 * int(key_heads) * key_dim + value_heads * value_dim, "x must hold the q, k and v channels")
    _require_cuda(a, "a", device)
    _require_cuda(b, "b", device)
    _require(a.shape == (batch, value_heads) and b.shape == (batch, value_heads), "a/b must be (batch, value_heads)")
    _require(a.dtype == b.dtype and a.dtype in (torch.float32, torch.bfloat16), "a/b must share a float32/bfloat16 dtype")
    a_c, b_c = a.contiguous(), b.contiguous()
    alog = _f32_contig(_flat(a_log), "a_log", device)
    dtb = _f32_contig(_flat(dt_bias), "dt_bias", device)
    slot_ptr, slot_code = 0, L.QA_I32
    if slots is not None:
        _require_cuda(slots, "slots", device)
        _index_dtype(slots, "slots")
        slots = slots.contiguous()
        slot_ptr, slot_code = _ptr(slots), _code(slots)
    z_ptr, z_code, z_sb, w_ptr, w_code = 0, L.QA_F32, 0, 0, L.QA_F32
    if z is not None:
        _require_cuda(z, "z", device)
        _float_dtype(z, "z")
        _require(norm_weight is not None, "the output stage needs norm_weight")
        zz = z if z.shape == (batch, value_heads * value_dim) else z.reshape(batch, value_heads * value_dim)
        _require(zz.stride(-1) == 1, "z rows must be contiguous")
        nw = _vector_on(norm_weight, device)
        _float_dtype(nw, "norm_weight")
        _require(nw.numel() == value_dim, "norm_weight must have value_dim elements")
        z_ptr, z_code, z_sb, w_ptr, w_code = _ptr(zz), _code(zz), zz.stride(0), _ptr(nw), _code(nw)
    else:
        _require(norm_weight is None, "norm_weight needs z")
    out = torch.empty((batch, value_heads, value_dim), dtype=out_dtype, device=device)
    status = lib.qa_gated_delta_step_conv(
        _ptr(x), _code(x), x.stride(0), _ptr(conv_state), channels * (kernel - 1), _ptr(w), kernel, _ptr(a_c), _ptr(b_c), _code(a_c),
        a_c.stride(0), _ptr(alog), _ptr(dtb), _ptr(state), state.stride(0), slot_ptr, slot_code, state.shape[0], z_ptr, z_code, z_sb, w_ptr,
        w_code, float(eps), _ptr(out), _code(out), out.stride(0), batch, int(key_heads), value_heads, key_dim, value_dim, _stream(device),
    )
    L.check(lib, status, "gated_delta_step_conv")
    return out


def chunk_gated_delta_rule(
    mixed_qkv: torch.Tensor,
    a: torch.Tensor,
    b: torch.Tensor,
    a_log: torch.Tensor,
    dt_bias: torch.Tensor,
    conv_weight: torch.Tensor,
    *,
    key_heads: int,
    value_heads: int,
    conv_state: torch.Tensor | None = None,
    initial_state: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.bfloat16,
    keep_conv_state: bool = True,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """Chunked prefill of a linear-attention layer from its raw projections.

    ``mixed_qkv`` ``(B, T, 2*Hqk*128 + Hv*128)`` (the ``in_proj_qkv`` output),
    ``a``/``b`` ``(B, T, Hv)``, ``a_log``/``dt_bias`` ``(Hv,)``, ``conv_weight``
    ``(C, 1, 4)`` or ``(C, 4)``.  Returns ``(core (B, T, Hv, 128), final_state
    (B, Hv, 128, 128) fp32, conv_state (B, C, 3) fp32 or None)``; ``core`` is
    the recurrence output before the gated RMSNorm
    (``src/reference_ops.py:240-283`` with the recurrence ``:291-322``).
    """
    lib = L.load_library()
    _require_cuda(mixed_qkv, "mixed_qkv")
    device = mixed_qkv.device
    _require(mixed_qkv.dtype == torch.bfloat16, "mixed_qkv must be bfloat16")
    _require(mixed_qkv.dim() == 3 and mixed_qkv.stride(-1) == 1, "mixed_qkv must be (batch, seq, channels) with contiguous channels")
    batch, seq, channels = mixed_qkv.shape
    dk = dv = 128
    _require(channels == 2 * key_heads * dk + value_heads * dv, "mixed_qkv channels must be 2*key_heads*128 + value_heads*128")
    _require_cuda(a, "a", device)
    _require_cuda(b, "b", device)
    _require(a.shape == (batch, seq, value_heads) and b.shape == a.shape, "a/b must be (batch, seq, value_heads)")
    _require(a.dtype == b.dtype and a.dtype in (torch.float32, torch.bfloat16), "a/b must share a float32/bfloat16 dtype")
    _require(a.stride() == b.stride() and a.stride(-1) == 1, "a/b must share strides with contiguous heads")
    alog = _f32_contig(_flat(a_log), "a_log", device)
    dtb = _f32_contig(_flat(dt_bias), "dt_bias", device)
    w = _conv_weight(conv_weight, channels, device)
    _require(w.shape[1] == 4, "conv kernel must be 4")
    conv_in = None
    if conv_state is not None:
        conv_in = _f32_contig(conv_state, "conv_state", device)
        _require(tuple(conv_in.shape) == (batch, channels, 3), "conv_state must be (batch, channels, 3)")
    state_in = None
    if initial_state is not None:
        state_in = _f32_contig(initial_state, "initial_state", device)
        _require(tuple(state_in.shape) == (batch, value_heads, dk, dv), "initial_state must be (batch, value_heads, 128, 128)")
    out = torch.empty((batch, seq, value_heads, dv), dtype=out_dtype, device=device)
    final = torch.empty((batch, value_heads, dk, dv), dtype=torch.float32, device=device)
    conv_out = torch.empty((batch, channels, 3), dtype=torch.float32, device=device) if keep_conv_state else None
    ws_bytes = lib.qa_chunk_gated_delta_workspace(batch, seq, int(key_heads), int(value_heads))
    workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
    status = lib.qa_chunk_gated_delta_rule(
        _ptr(mixed_qkv), _code(mixed_qkv), mixed_qkv.stride(0), mixed_qkv.stride(1), _ptr(a), _ptr(b), _code(a), a.stride(0), a.stride(1),
        _ptr(alog), _ptr(dtb), _ptr(w), _ptr(conv_in), _ptr(conv_out), _ptr(state_in), _ptr(final), _ptr(out), _code(out), out.stride(0),
        out.stride(1), batch, seq, int(key_heads), int(value_heads), dk, dv, 4, _ptr(workspace), ws_bytes, _stream(device),
    )
    L.check(lib, status, "chunk_gated_delta_rule")
    return out, final, conv_out


def gated_rms_norm(core: torch.Tensor, z: torch.Tensor, weight: torch.Tensor, eps: float, *, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """The output stage of a linear-attention layer: gated RMSNorm + SiLU(z) per value head.

    ``core`` ``(..., heads, head_dim)`` (the recurrence output, float32 or bfloat16; its
    ``head_dim`` axis contiguous), ``z`` the ``in_proj_z`` output ``(..., heads * head_dim)`` or
    ``(..., heads, head_dim)``, ``weight`` ``(head_dim,)``.  Returns ``(..., heads * head_dim)``
    in ``out_dtype`` (default: ``core``'s dtype, as ``gated_rms_norm`` returns,
    ``src/reference_ops.py:172-178,284-287``).
    """
    lib = L.load_library()
    _require_cuda(core, "core")
    device = core.device
    _require_cuda(z, "z", device)
    _float_dtype(core, "core")
    _float_dtype(z, "z")
    _require(core.dim() >= 2 and core.stride(-1) == 1, "core must be (..., heads, head_dim) with a contiguous head_dim axis")
    heads, head_dim = core.shape[-2], core.shape[-1]
    lead = core.shape[:-2]
    x = core.reshape(-1, heads, head_dim)
    gate = z.reshape(*lead, heads, head_dim).reshape(-1, heads, head_dim)
    _require(gate.stride(-1) == 1, "z must have a contiguous head_dim axis")
    w = _vector_on(weight, device)
    _float_dtype(w, "weight")
    _require(w.numel() == head_dim, "weight must have head_dim elements")
    out = torch.empty((x.shape[0], heads, head_dim), dtype=out_dtype or core.dtype, device=device)
    _float_dtype(out, "out")
    status = lib.qa_gated_rms_norm(
        _ptr(x), _code(x), x.stride(0), x.stride(1), _ptr(gate), _code(gate), gate.stride(0), gate.stride(1), _ptr(w), _code(w), float(eps),
        x.shape[0], int(heads), int(head_dim), _ptr(out), _code(out), out.stride(0), out.stride(1), _stream(device),
    )
    L.check(lib, status, "gated_rms_norm")
    return out.reshape(*lead, heads * head_dim)


def paged_attention_prefill(
    query: torch.Tensor,
    cu_seqlens: torch.Tensor,
    prefix_lens: torch.Tensor,
    key_pool: torch.Tensor,
    value_pool: torch.Tensor,
    block_tables: torch.Tensor,
    block_size: int,
    *,
    max_new: int,
    gate: torch.Tensor | None = None,
    scale: float | None = None,
) -> torch.Tensor:
    """Causal attention of packed new tokens over the shared paged pool, with optional gate.

    ``query`` ``(total_new, H, D)`` bf16; ``cu_seqlens`` ``(B+1,)`` and
    ``prefix_lens`` ``(B,)`` device index arrays; the new tokens' K/V must
    already be appended to ``key_pool``/``value_pool`` ``(P, H_kv, bs, D)`` at
    positions ``prefix_b + n``.  ``gate`` ``(total_new, H*D)`` bf16 logits, or a
    ``(total_new, H, D)`` view with a contiguous last dimension (such as the second half of
    each ``q_proj`` head, read in place), give ``out * sigmoid(gate)``
    (``src/reference_ops.py:338-340,360``).  Returns
    ``(total_new, H, D)`` bf16.
    """
    lib = L.load_library()
    _require_cuda(query, "query")
    device = query.device
    _require(query.dtype == torch.bfloat16 and query.dim() == 3 and query.stride(-1) == 1, "query must be (tokens, heads, head_dim) bfloat16")
    for tensor, name in ((cu_seqlens, "cu_seqlens"), (prefix_lens, "prefix_lens"), (block_tables, "block_tables")):
        _require_cuda(tensor, name, device)
        _index_dtype(tensor, name)
    _require(cu_seqlens.dtype == prefix_lens.dtype, "cu_seqlens and prefix_lens must share a dtype")
    _require(key_pool.dim() == 4, "prefill needs a shared pool (blocks, kv_heads, block_size, head_dim)")
    desc = _pool_descriptor(key_pool, value_pool, "shared")
    batch = prefix_lens.shape[0]
    _require(cu_seqlens.shape[0] == batch + 1, "cu_seqlens must have batch + 1 entries")
    tokens, heads, head_dim = query.shape
    gate_c = None
    gate_sh = 0
    if gate is not None:
        _require_cuda(gate, "gate", device)
        _require(gate.dtype == torch.bfloat16, "gate must be bfloat16")
        if gate.dim() == 3:  # (tokens, heads, head_dim) view, e.g. the second half of each q_proj head
            _require(gate.shape == (tokens, heads, head_dim), "gate must be (tokens, heads*head_dim) or (tokens, heads, head_dim)")
            gate_c = gate if gate.stride(-1) == 1 else gate.contiguous()
            gate_sh = gate_c.stride(1)
        else:
            _require(gate.shape == (tokens, heads * head_dim), "gate must be (tokens, heads*head_dim) or (tokens, heads, head_dim)")
            gate_c = gate.contiguous()
    tables = block_tables.contiguous()
    out = torch.empty((tokens, heads, head_dim), dtype=torch.bfloat16, device=device)
    status = lib.qa_paged_attention_prefill(
        _ptr(query), _code(query), query.stride(0), query.stride(1), _ptr(cu_seqlens.contiguous()), _ptr(prefix_lens.contiguous()),
        _code(cu_seqlens), batch, int(max_new), heads, head_dim, ctypes.byref(desc), _ptr(tables), _code(tables), tables.stride(0),
        tables.shape[1], int(block_size), float(scale or 0.0), _ptr(gate_c), 0 if gate_c is None else gate_c.stride(0), gate_sh, _ptr(out),
        _stream(device),
    )
    L.check(lib, status, "paged_attention_prefill")
    return out


_INV_FREQ: dict[tuple[int, float, torch.device], torch.Tensor] = {}


def rope_inv_freq(rotary_dim: int, rope_theta: float, device: torch.device) -> torch.Tensor:
    """``inv_freq`` of ``rotary_embeddings`` (``src/reference_ops.py:203-213``), computed as the
    reference computes it (fp32 torch on the CPU), moved to ``device`` once per
    (rotary_dim, theta, device)."""
    key = (int(rotary_dim), float(rope_theta), device)
    cached = _INV_FREQ.get(key)
    if cached is None:
        inv = 1.0 / (float(rope_theta) ** (torch.arange(0, rotary_dim, 2, dtype=torch.float32) / rotary_dim))
        cached = inv.to(device)
        _INV_FREQ[key] = cached
    return cached


_COS_SIN: dict[tuple[int, float, torch.device], torch.Tensor] = {}


def rope_cos_sin_table(rotary_dim: int, rope_theta: float, positions: int, device: torch.device) -> torch.Tensor:
    """bf16 ``(positions, 2, rotary_dim/2)`` cos and sin of ``pos * inv_freq``, computed with the
    torch CPU operations of ``rotary_embeddings`` (``src/reference_ops.py:203-213``: fp32 angles,
    fp32 cos/sin, cast to bf16) so the values are the reference's bit for bit; cached per
    (rotary_dim, theta, device) and regrown when more positions are asked for."""
    key = (int(rotary_dim), float(rope_theta), device)
    cached = _COS_SIN.get(key)
    if cached is None or cached.shape[0] < positions:
        freqs = torch.outer(torch.arange(positions, dtype=torch.float32), rope_inv_freq(rotary_dim, rope_theta, torch.device("cpu")))
        table = torch.stack((freqs.cos(), freqs.sin()), dim=1).to(torch.bfloat16).contiguous()
        cached = table.to(device)
        _COS_SIN[key] = cached
    return cached


def qk_norm_rope_kv_append(
    q_proj: torch.Tensor,
    k_proj: torch.Tensor,
    v_proj: torch.Tensor,
    q_norm_weight: torch.Tensor,
    k_norm_weight: torch.Tensor,
    key_pool: torch.Tensor,
    value_pool: torch.Tensor,
    block_tables: torch.Tensor,
    cu_seqlens: torch.Tensor,
    starts: torch.Tensor,
    block_size: int,
    *,
    max_new: int,
    eps: float,
    rope_theta: float,
    partial_rotary_factor: float,
    table_positions: int = 131072,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Prologue of a full-attention layer over packed new tokens, in one launch.

    ``q_proj`` ``(tokens, H, 2D)`` (or ``(tokens, H*2D)``), ``k_proj``/``v_proj`` ``(tokens, H_kv, D)``
    (or ``(tokens, H_kv*D)``), bf16, as the projections produce them; row ``b`` owns tokens
    ``cu_seqlens[b]:cu_seqlens[b+1]`` at positions ``starts[b] + n``.  Applies the reference's
    ``rms_norm`` with the ``(1 + w)`` weight and ``apply_rotary_pos_emb`` with
    ``rotary_dim = int(D * partial_rotary_factor)`` (``src/reference_ops.py:343-347``,
    ``src/tp_runtime.py:511-525``), appends k and v to the shared pool ``(P, H_kv, bs, D)`` at
    those positions (the reference's ``cache.append``, ``src/decode_state.py:271-293``, without
    repeating heads), and returns ``(query (tokens, H, D) bf16, gate (tokens, H, D) view of
    q_proj)`` ready for :func:`paged_attention_prefill` or, for one token per row, decode.
    The bf16 cos/sin of positions below ``table_positions`` come from :func:`rope_cos_sin_table`;
    the kernel computes those of later positions itself.
    """
    lib = L.load_library()
    _require_cuda(q_proj, "q_proj")
    device = q_proj.device
    for tensor, name in ((k_proj, "k_proj"), (v_proj, "v_proj"), (q_norm_weight, "q_norm_weight"), (k_norm_weight, "k_norm_weight"),
                         (key_pool, "key_pool"), (value_pool, "value_pool"), (block_tables, "block_tables"), (cu_seqlens, "cu_seqlens"),
                         (starts, "starts")):
        _require_cuda(tensor, name, device)
    _require(key_pool.dim() == 4, "qk_norm_rope_kv_append needs a shared pool (blocks, kv_heads, block_size, head_dim)")
    _, kv_heads, _, head_dim = key_pool.shape
    tokens = q_proj.shape[0]
    q3 = q_proj.view(tokens, -1, 2 * head_dim) if q_proj.dim() == 2 else q_proj
    k3 = k_proj.view(tokens, kv_heads, head_dim) if k_proj.dim() == 2 else k_proj
    v3 = v_proj.view(tokens, kv_heads, head_dim) if v_proj.dim() == 2 else v_proj
    heads = q3.shape[1]
    _require(q3.dim() == 3 and q3.shape[2] == 2 * head_dim, "q_proj must be (tokens, heads, 2*head_dim)")
    _require(k3.shape == (tokens, kv_heads, head_dim) and v3.shape == (tokens, kv_heads, head_dim), "k_proj/v_proj must be (tokens, kv_heads, head_dim)")
    for tensor, name in ((q3, "q_proj"), (k3, "k_proj"), (v3, "v_proj"), (key_pool, "key_pool")):
        if tensor.dtype != torch.bfloat16 or tensor.stride(-1) != 1:
            raise RuntimeError(f"{name} must be bfloat16 with a contiguous last dimension")
    _float_dtype(q_norm_weight, "q_norm_weight")
    _require(q_norm_weight.dtype == k_norm_weight.dtype and q_norm_weight.shape == (head_dim,) and k_norm_weight.shape == (head_dim,),
             "norm weights must be (head_dim,) of one dtype")
    for tensor, name in ((cu_seqlens, "cu_seqlens"), (starts, "starts"), (block_tables, "block_tables")):
        _index_dtype(tensor, name)
    _require(cu_seqlens.dtype == starts.dtype, "cu_seqlens and starts must share a dtype")
    batch = starts.shape[0]
    _require(cu_seqlens.shape[0] == batch + 1, "cu_seqlens must have batch + 1 entries")
    tables = block_tables.contiguous() if block_tables.dim() == 2 else block_tables.contiguous().view(1, -1).expand(batch, -1)
    rotary_dim = int(head_dim * partial_rotary_factor)
    inv_freq = rope_inv_freq(rotary_dim, rope_theta, device)
    cos_sin = rope_cos_sin_table(rotary_dim, rope_theta, int(table_positions), device) if rotary_dim > 0 and table_positions > 0 else None
    qw = q_norm_weight.contiguous()
    kw = k_norm_weight.contiguous()
    desc = _pool_descriptor(key_pool, value_pool, "shared")
    query = torch.empty((tokens, heads, head_dim), dtype=torch.bfloat16, device=device)
    status = lib.qa_qk_norm_rope_append(
        _ptr(q3), q3.stride(0), q3.stride(1), _ptr(k3), k3.stride(0), k3.stride(1), _ptr(v3), v3.stride(0), v3.stride(1), _code(q3),
        _ptr(qw), _ptr(kw), _code(qw), float(eps), _ptr(inv_freq), _ptr(cos_sin), 0 if cos_sin is None else cos_sin.shape[0], rotary_dim,
        _ptr(cu_seqlens.contiguous()), _ptr(starts.contiguous()),
        _code(cu_seqlens), batch, int(max_new), heads, head_dim, ctypes.byref(desc), _ptr(tables), _code(tables), tables.stride(0),
        tables.shape[1], int(block_size), _ptr(query), _stream(device),
    )
    L.check(lib, status, "qk_norm_rope_kv_append")
    return query, q3.narrow(2, head_dim, head_dim)


# --------------------------------------------------------------------------- the 4-bit KV cache


def _launch(device: torch.device, fn: Any, *args: Any) -> int:
    """``fn(*args, stream)`` on ``device``'s current stream, with that device current."""
    index = device.index
    if torch._C._cuda_getDevice() == index:
        return fn(*args, torch._C._cuda_getCurrentRawStream(index))
    with torch.cuda.device(device):
        return fn(*args, torch._C._cuda_getCurrentRawStream(index))


def _same_device(device: torch.device, **tensors: Any) -> None:
    """Names the tensor that is not on ``device`` (called where a cheaper check has found one)."""
    for name, tensor in tensors.items():
        _require_cuda(tensor, name, device)


def kv4_tile_bytes(head_dim: int, block_size: int) -> int:
    """Bytes of one block of one KV head in a 4-bit pool: 4 bits a value and a scale byte per 32 values."""
    _require(head_dim in (128, 256), "4-bit pools need head_dim 128 or 256")
    _require(16 <= block_size <= 1024 and block_size & (block_size - 1) == 0, "4-bit pools need a block_size that is a power of two from 16 to 1024")
    return block_size * 17 * head_dim // 32


def _kv4_descriptor(key_pool: torch.Tensor, value_pool: torch.Tensor, block_size: int, device: torch.device) -> tuple[L.PagedKV, int]:
    """Descriptor and head_dim of a 4-bit pool ``(P, H_kv, kv4_tile_bytes(D, block_size))``."""
    if key_pool.device != device or value_pool.device != device:
        _same_device(device, key_pool=key_pool, value_pool=value_pool)
    shape, strides = key_pool.shape, key_pool.stride()
    if key_pool.dtype is not torch.uint8 or value_pool.dtype is not torch.uint8 or len(shape) != 3 or value_pool.shape != shape:
        raise RuntimeError("4-bit pools must be uint8 (blocks, kv_heads, tile bytes) and alike")
    if strides[2] != 1 or value_pool.stride() != strides:
        raise RuntimeError("key/value pools must share strides with contiguous tiles")
    blocks, kv_heads, tile = shape
    for head_dim in (256, 128):
        if tile * 32 == block_size * 17 * head_dim:
            return L.PagedKV(key_pool.data_ptr(), value_pool.data_ptr(), None, None, None, blocks, 0, strides[0], strides[1], 0, kv_heads, L.QA_KV4), head_dim
    raise RuntimeError(f"a tile of {tile} bytes is no block of {block_size} tokens of 128 or 256 dims in 4 bits")


def _rows(tensor: torch.Tensor, multiple: int) -> tuple[torch.Tensor, int, int]:
    """``tensor`` (.., .., D) as it is where its rows can be read in aligned pieces of ``multiple`` elements, else a
    copy; and its row strides."""
    strides = tensor.stride()
    if strides[-1] == 1 and strides[0] % multiple == 0 and strides[1] % multiple == 0 and tensor.data_ptr() % (multiple * tensor.element_size()) == 0:
        return tensor, strides[0], strides[1]
    # not .contiguous(): it gives back a contiguous tensor at an odd address, or a single row of an odd stride, as it is
    tensor = tensor.clone(memory_format=torch.contiguous_format)
    strides = tensor.stride()
    return tensor, strides[0], strides[1]


def _kv4_gate(gate: torch.Tensor | None, rows: int, heads: int, head_dim: int, device: torch.device) -> tuple[torch.Tensor | None, int, int, int]:
    """The gate as ``(tensor to keep, pointer, token stride, head stride)``."""
    if gate is None:
        return None, 0, 0, 0
    if gate.device != device:
        _require_cuda(gate, "gate", device)
    _require(gate.dtype is torch.bfloat16, "gate must be bfloat16")
    if gate.dim() == 2 and gate.shape == (rows, heads * head_dim):
        gate = gate.reshape(rows, heads, head_dim)
    _require(gate.shape == (rows, heads, head_dim), "gate must be (tokens, heads*head_dim) or (tokens, heads, head_dim)")
    gate, stride_t, stride_h = _rows(gate, 4)
    return gate, gate.data_ptr(), stride_t, stride_h


def _kv4_out(out: torch.Tensor | None, like: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty_like(like) if like.is_contiguous() else like.new_empty(like.shape)
    _require_cuda(out, "out", like.device)
    _require(out.dtype == torch.bfloat16 and out.shape == like.shape and out.is_contiguous(), "out must be contiguous bfloat16 of query's shape")
    return out


class PagedPlan(NamedTuple):
    """A step of packed new tokens on the device (:func:`paged_kv_plan`): ``cu_seqlens`` ``(B + 1,)`` and ``starts``
    ``(B,)`` int32 (each row's tokens and its length before the step), ``positions`` int32 and ``slots`` int64
    ``(max_tokens,)``, -1 past the step's last token."""

    cu_seqlens: torch.Tensor
    starts: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor


class PagedStepPlan(PagedPlan):
    """The plan of a decode step, one entry a row (``DeviceBatchPageTables.plan_step``).  ``lengths`` ``(B,)`` int32 are
    what the step's attention reads: a row's tokens with its new one, 0 where it takes none, so that a row without a
    request, and every row of a step that was refused, gives zeros."""

    lengths: torch.Tensor

    @classmethod
    def of(cls, plan: PagedPlan) -> "PagedStepPlan":
        step = cls(*plan)
        step.lengths = plan.positions + 1  # -1 where there is no new token
        return step


def paged_kv_plan(
    block_tables: torch.Tensor,
    lengths: torch.Tensor,
    counts: torch.Tensor | int,
    free_list: torch.Tensor,
    free_state: torch.Tensor,
    status: torch.Tensor,
    block_size: int,
    *,
    max_tokens: int,
    per_row: int = 0,
) -> PagedPlan:
    """Block tables and slot map of a batched step, built on the device from the requests' lengths.

    Row ``b`` grows from ``lengths[b]`` to ``lengths[b] + counts_b`` tokens: fresh logical blocks get ids from the
    front of the ascending ``free_list``, rows in order (:func:`paged_kv_reserve`'s policy), and ``block_tables``
    ``(B, max_blocks)`` int32, ``lengths`` ``(B,)`` int32 and ``free_state`` are advanced in place.  The returned
    plan holds the packed step for :func:`qk_norm_mrope_kv_append`, :func:`paged_kv4_append` and
    :func:`paged_attention_prefill_kv4`.  ``max_tokens`` bounds the step (the host need not know its size), and the
    token arrays are that long.  ``status`` (int32 ``[1]``) becomes 0, or 1 (pool exhausted), 2 (a table row too
    short), 3 (corrupt free state), 4 (negative or overflowing length or count), 5 (more than ``max_tokens``
    tokens): then nothing is taken and the plan is empty.  Operators fed by its slots and ``cu_seqlens`` write nothing
    to the pool and compute no token; a decode takes ``positions + 1`` as its lengths (``lengths`` are the rows' old
    ones) and gives zeros.  The next plan overwrites ``status``, so it has to be read before that.  Nothing is read
    back here, so the call can be captured in a HIP graph.

    With ``per_row`` the token arrays are not packed but hold ``per_row`` entries for each row (``max_tokens`` is
    ``B * per_row``), a row's tokens first and -1 behind them: the form of a decode step, whose operators take one
    token of every row whether it holds a request or not.
    """
    lib = L.load_library()
    device = block_tables.device
    if device.type != "cuda" or not (lengths.device == free_list.device == free_state.device == status.device == device):
        _same_device(device, block_tables=block_tables, lengths=lengths, free_list=free_list, free_state=free_state, status=status)
    i32 = torch.int32
    _require(block_tables.dtype is i32 and block_tables.dim() == 2 and block_tables.stride(1) == 1, "block_tables must be int32 [batch, max_blocks] with contiguous rows")
    batch, max_blocks = block_tables.shape
    _require(batch > 0 and max_blocks > 0, "block_tables must have shape [batch, max_blocks]")
    _require(lengths.dtype is i32 and lengths.shape == (batch,) and lengths.is_contiguous(), "lengths must be a contiguous int32 [batch] tensor")
    _require(free_list.dtype is i32 and free_list.dim() == 1 and free_list.is_contiguous(), "free_list must be a contiguous int32 vector")
    _require(free_state.dtype is i32 and free_state.numel() == 2 and free_state.is_contiguous(), "free_state must be int32 [head, count]")
    _require(status.dtype is i32 and status.numel() >= 1, "status must be an int32 tensor")
    max_tokens = int(max_tokens)
    per_row = int(per_row)
    _require(max_tokens >= 0, "max_tokens must be non-negative")
    _require(per_row == 0 or per_row * batch == max_tokens, "with per_row entries a row max_tokens must be batch * per_row")
    count_ptr, count_code, count_scalar = 0, L.QA_I32, 0
    if isinstance(counts, torch.Tensor):
        if counts.device != device:
            _require_cuda(counts, "counts", device)
        _index_dtype(counts, "counts")
        _require(counts.shape == (batch,) and counts.is_contiguous(), "counts must be a contiguous [batch] tensor")
        count_ptr, count_code = counts.data_ptr(), _code(counts)
    else:
        count_scalar = int(counts)
        _require(count_scalar >= 0, "counts must be non-negative")
    slots = torch.empty(max_tokens, dtype=torch.int64, device=device)
    # one allocation: cu_seqlens, starts, the kernel's scratch row sums, positions
    ints = lengths.new_empty(3 * batch + 1 + max_tokens)
    at = ints.data_ptr()
    code = _launch(
        device, lib.qa_paged_kv_plan, block_tables.data_ptr(), block_tables.stride(0), max_blocks, lengths.data_ptr(), count_ptr, count_code, count_scalar, batch,
        int(block_size), free_list.data_ptr(), free_list.numel(), free_state.data_ptr(), status.data_ptr(), max_tokens, per_row, at, at + 4 * (batch + 1), at + 4 * (3 * batch + 1),
        slots.data_ptr(), at + 4 * (2 * batch + 1), 4 * batch,
    )
    L.check(lib, code, "paged_kv_plan")
    cu_seqlens, starts, _, positions = ints.split_with_sizes((batch + 1, batch, batch, max_tokens))
    return PagedPlan(cu_seqlens, starts, positions, slots)


def _tiles_append(what: str, descriptor: Any, key: torch.Tensor, value: torch.Tensor, key_pool: torch.Tensor, value_pool: torch.Tensor, slots: torch.Tensor, block_size: int) -> None:
    """``paged_kv4_append`` and ``paged_kv8_append``: the operator of a pool of tiles in 4 or 8 bits; ``descriptor`` checks the pool."""
    lib = L.load_library()
    device = key.device
    if device.type != "cuda" or not (value.device == slots.device == device):
        _same_device(device, key=key, value=value, slots=slots)
    _index_dtype(slots, "slots")
    desc, head_dim = descriptor(key_pool, value_pool, block_size, device)
    shape = key.shape
    _require(len(shape) == 3 and shape[1] == desc.kv_heads and shape[2] == head_dim and value.shape == shape, "key/value must be (tokens, kv_heads, head_dim) of the pool's heads")
    _float_dtype(key, "key")
    _require(value.dtype is key.dtype, "key and value must share a dtype")
    _require(slots.shape == shape[:1], "slots must have one entry per token")
    multiple = 8 if key.dtype is torch.bfloat16 else 4
    k, k_st, k_sh = _rows(key, multiple)
    v, v_st, v_sh = _rows(value, multiple)
    s = slots.contiguous()
    code = _launch(
        device, getattr(lib, f"qa_{what}"), k.data_ptr(), v.data_ptr(), _code(k), k_st, k_sh, v_st, v_sh, shape[0], head_dim, ctypes.byref(desc), s.data_ptr(), _code(s),
        int(block_size),
    )
    L.check(lib, code, what)


def _tiles_gather(what: str, descriptor: Any, key_pool: torch.Tensor, value_pool: torch.Tensor, block_tables: torch.Tensor, valid: int, block_size: int) -> tuple[torch.Tensor, torch.Tensor]:
    """``paged_kv4_gather`` and ``paged_kv8_gather``: the operator of a pool of tiles in 4 or 8 bits; ``descriptor`` checks the pool."""
    lib = L.load_library()
    device = key_pool.device
    if device.type != "cuda" or block_tables.device != device:
        _same_device(device, key_pool=key_pool, block_tables=block_tables)
    _index_dtype(block_tables, "block_tables")
    desc, head_dim = descriptor(key_pool, value_pool, block_size, device)
    tables = block_tables.contiguous()
    if tables.dim() == 1:
        tables = tables.unsqueeze(0)
    _require(tables.dim() == 2 and tables.shape[1] > 0, "block_tables must have shape [batch, max_blocks]")
    batch, max_blocks = tables.shape
    valid = int(valid)
    _require(valid >= 0, "valid must be non-negative")
    key_out = torch.empty((batch, desc.kv_heads, valid, head_dim), dtype=torch.bfloat16, device=device)
    value_out = torch.empty_like(key_out)
    code = _launch(
        device, getattr(lib, f"qa_{what}"), ctypes.byref(desc), head_dim, batch, tables.data_ptr(), _code(tables), max_blocks, max_blocks, valid, int(block_size),
        key_out.data_ptr(), value_out.data_ptr(),
    )
    L.check(lib, code, what)
    return key_out, value_out


def _tiles_decode(
    what: str, descriptor: Any, query: torch.Tensor, block_tables: torch.Tensor, key_pool: torch.Tensor, value_pool: torch.Tensor, sequence_lengths: torch.Tensor, block_size: int,
    gate: torch.Tensor | None, scale: float | None, out: torch.Tensor | None,
) -> torch.Tensor:
    """``paged_attention_decode_kv4`` and ``paged_attention_decode_kv8``: the operator of a pool of tiles in 4 or 8 bits; ``descriptor`` checks the pool."""
    lib = L.load_library()
    device = query.device
    if device.type != "cuda" or not (block_tables.device == sequence_lengths.device == device):
        _same_device(device, query=query, block_tables=block_tables, sequence_lengths=sequence_lengths)
    _require(query.dtype is torch.bfloat16, "query must be bfloat16")
    _index_dtype(block_tables, "block_tables")
    _index_dtype(sequence_lengths, "sequence_lengths")
    shape = query.shape
    _require(len(shape) == 4 and shape[2] == 1, "query must have shape [batch, heads, 1, head_dim]")
    desc, head_dim = descriptor(key_pool, value_pool, block_size, device)
    batch, heads = shape[0], shape[1]
    _require(shape[3] == head_dim, "KV head_dim must match query")
    _require(block_tables.dim() == 2 and block_tables.shape[0] == batch and block_tables.shape[1] > 0, "block_tables must have shape [batch, max_blocks]")
    _require(sequence_lengths.shape == shape[:1], "sequence_lengths batch must match query")
    _require(heads % desc.kv_heads == 0, "KV heads must divide query heads")
    q, q_sb, q_sh = _rows(query, 8)
    g, g_ptr, g_sb, g_sh = _kv4_gate(gate, batch, heads, head_dim, device)
    tables, lens = block_tables.contiguous(), sequence_lengths.contiguous()
    max_blocks = tables.shape[1]
    result = _kv4_out(out, query)
    nbytes = getattr(lib, f"qa_{what}_workspace")(batch, heads, desc.kv_heads, head_dim, max_blocks * block_size)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    code = _launch(
        device, getattr(lib, f"qa_{what}"), q.data_ptr(), L.QA_BF16, q_sb, q_sh, batch, heads, head_dim, ctypes.byref(desc), tables.data_ptr(), _code(tables),
        max_blocks, max_blocks, lens.data_ptr(), _code(lens), int(block_size), float(scale or 0.0), g_ptr, g_sb, g_sh, result.data_ptr(), _ptr(ws), nbytes,
    )
    L.check(lib, code, what)
    return result


def _tiles_prefill(
    what: str, descriptor: Any, query: torch.Tensor, cu_seqlens: torch.Tensor, prefix_lens: torch.Tensor, key_pool: torch.Tensor, value_pool: torch.Tensor, block_tables: torch.Tensor,
    block_size: int, max_new: int, gate: torch.Tensor | None, scale: float | None, out: torch.Tensor | None,
) -> torch.Tensor:
    """``paged_attention_prefill_kv4`` and ``paged_attention_prefill_kv8``: the operator of a pool of tiles in 4 or 8 bits; ``descriptor`` checks the pool."""
    lib = L.load_library()
    device = query.device
    if device.type != "cuda" or not (cu_seqlens.device == prefix_lens.device == block_tables.device == device):
        _same_device(device, query=query, cu_seqlens=cu_seqlens, prefix_lens=prefix_lens, block_tables=block_tables)
    shape = query.shape
    _require(query.dtype is torch.bfloat16 and len(shape) == 3, "query must be (tokens, heads, head_dim) bfloat16")
    _index_dtype(cu_seqlens, "cu_seqlens")
    _index_dtype(block_tables, "block_tables")
    _require(cu_seqlens.dtype is prefix_lens.dtype, "cu_seqlens and prefix_lens must share a dtype")
    desc, head_dim = descriptor(key_pool, value_pool, block_size, device)
    tokens, heads = shape[0], shape[1]
    _require(shape[2] == head_dim, "KV head_dim must match query")
    _require(heads % desc.kv_heads == 0, "KV heads must divide query heads")
    _require(prefix_lens.dim() == 1 and cu_seqlens.shape == (prefix_lens.shape[0] + 1,), "cu_seqlens must have batch + 1 entries")
    batch = prefix_lens.shape[0]
    _require(block_tables.dim() == 2 and block_tables.shape[0] == batch and block_tables.shape[1] > 0, "block_tables must have shape [batch, max_blocks]")
    q, q_st, q_sh = _rows(query, 8)
    g, g_ptr, g_st, g_sh = _kv4_gate(gate, tokens, heads, head_dim, device)
    cu, prefix, tables = cu_seqlens.contiguous(), prefix_lens.contiguous(), block_tables.contiguous()
    max_blocks = tables.shape[1]
    result = _kv4_out(out, query)
    nbytes = getattr(lib, f"qa_{what}_workspace")(tokens, batch, int(max_new), heads, desc.kv_heads, head_dim, max_blocks * block_size)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    code = _launch(
        device, getattr(lib, f"qa_{what}"), q.data_ptr(), L.QA_BF16, q_st, q_sh, tokens, cu.data_ptr(), prefix.data_ptr(), _code(cu), batch, int(max_new),
        heads, head_dim, ctypes.byref(desc), tables.data_ptr(), _code(tables), max_blocks, max_blocks, int(block_size), float(scale or 0.0), g_ptr, g_st, g_sh,
        result.data_ptr(), _ptr(ws), nbytes,
    )
    L.check(lib, code, what)
    return result


def paged_kv4_append(key: torch.Tensor, value: torch.Tensor, key_pool: torch.Tensor, value_pool: torch.Tensor, slots: torch.Tensor, block_size: int) -> None:
    """Quantise packed K/V rows ``(tokens, H_kv, D)`` (bf16 or fp32) into ``slots`` of a 4-bit pool, in place.

    The pools are uint8 ``(P, H_kv, kv4_tile_bytes(D, block_size))``; per 32 dims of a token a power-of-two scale and
    E2M1 codes (the format and layout stand in ``qwen36_hip.h``).  ``slots`` ``(tokens,)`` hold ``block id *
    block_size + position % block_size`` (:func:`paged_kv_plan`); those outside the pool, such as -1, are skipped.
    They have to be distinct.
    """
    _tiles_append("paged_kv4_append", _kv4_descriptor, key, value, key_pool, value_pool, slots, block_size)


def paged_kv4_gather(key_pool: torch.Tensor, value_pool: torch.Tensor, block_tables: torch.Tensor, valid: int, block_size: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Dense ``(B, H_kv, valid, D)`` bf16 K/V of a 4-bit pool in logical order (:func:`paged_kv_gather`'s counterpart).

    Every value the cache holds is exact in bf16.  Tokens whose block id is outside the pool, or past the table, are
    zeros; a group stored from an infinity or a NaN reads as NaN.
    """
    return _tiles_gather("paged_kv4_gather", _kv4_descriptor, key_pool, value_pool, block_tables, valid, block_size)


def paged_attention_decode_kv4(
    query: torch.Tensor,
    block_tables: torch.Tensor,
    key_pool: torch.Tensor,
    value_pool: torch.Tensor,
    sequence_lengths: torch.Tensor,
    block_size: int,
    *,
    gate: torch.Tensor | None = None,
    scale: float | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``paged_attention_decode_batched`` over a 4-bit pool: one token per row, ``query`` ``(B, H, 1, D)`` bf16.

    ``gate`` ``(B, H*D)`` or ``(B, H, D)`` bf16 logits (a view of ``q_proj`` is read in place) give ``out *
    sigmoid(gate)``.  Rows of length <= 0, and rows that see only blocks outside the pool, give zeros.  Returns
    ``(B, H, 1, D)`` bf16, in ``out`` where it is given.
    """
    return _tiles_decode("paged_attention_decode_kv4", _kv4_descriptor, query, block_tables, key_pool, value_pool, sequence_lengths, block_size, gate, scale, out)


def paged_attention_prefill_kv4(
    query: torch.Tensor,
    cu_seqlens: torch.Tensor,
    prefix_lens: torch.Tensor,
    key_pool: torch.Tensor,
    value_pool: torch.Tensor,
    block_tables: torch.Tensor,
    block_size: int,
    *,
    max_new: int,
    gate: torch.Tensor | None = None,
    scale: float | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """:func:`paged_attention_prefill` over a 4-bit pool: causal attention of packed new tokens.

    ``query`` ``(tokens, H, D)`` bf16; the new tokens' K/V are in the pool already, so a new token sees itself and
    its neighbours in 4 bits, as every later step will.  ``max_new`` is at least the longest row of ``cu_seqlens``
    (tokens past it are not computed).  Returns ``(tokens, H, D)`` bf16, in ``out`` where it is given; rows past the
    last sequence are not written.
    """
    return _tiles_prefill("paged_attention_prefill_kv4", _kv4_descriptor, query, cu_seqlens, prefix_lens, key_pool, value_pool, block_tables, block_size, max_new, gate, scale, out)


def kv8_tile_bytes(head_dim: int, block_size: int) -> int:
    """Bytes of one block of one KV head in an 8-bit pool: 8 bits a value, and 16 bytes per 16 tokens for their scale."""
    _require(head_dim in (128, 256), "8-bit pools need head_dim 128 or 256")
    _require(16 <= block_size <= 1024 and block_size & (block_size - 1) == 0, "8-bit pools need a block_size that is a power of two from 16 to 1024")
    return block_size * (head_dim + 1)


def _kv8_descriptor(key_pool: torch.Tensor, value_pool: torch.Tensor, block_size: int, device: torch.device) -> tuple[L.PagedKV, int]:
    """Descriptor and head_dim of an 8-bit pool ``(P, H_kv, kv8_tile_bytes(D, block_size))``."""
    if key_pool.device != device or value_pool.device != device:
        _same_device(device, key_pool=key_pool, value_pool=value_pool)
    shape, strides = key_pool.shape, key_pool.stride()
    if key_pool.dtype is not torch.float8_e4m3fn or value_pool.dtype is not torch.float8_e4m3fn or len(shape) != 3 or value_pool.shape != shape:
        raise RuntimeError("8-bit pools must be float8_e4m3fn (blocks, kv_heads, tile bytes) and alike")
    if strides[2] != 1 or value_pool.stride() != strides:
        raise RuntimeError("key/value pools must share strides with contiguous tiles")
    blocks, kv_heads, tile = shape
    for head_dim in (256, 128):
        if tile == block_size * (head_dim + 1):
            return L.PagedKV(key_pool.data_ptr(), value_pool.data_ptr(), None, None, None, blocks, 0, strides[0], strides[1], 0, kv_heads, L.QA_KV8), head_dim
    raise RuntimeError(f"a tile of {tile} bytes is no block of {block_size} tokens of 128 or 256 dims in 8 bits")


def paged_kv8_append(key: torch.Tensor, value: torch.Tensor, key_pool: torch.Tensor, value_pool: torch.Tensor, slots: torch.Tensor, block_size: int) -> None:
    """Quantise packed K/V rows ``(tokens, H_kv, D)`` (bf16 or fp32) into ``slots`` of an 8-bit pool, in place.

    The pools are float8_e4m3fn ``(P, H_kv, kv8_tile_bytes(D, block_size))``: E4M3 codes, and a power-of-two scale for each run of
    16 tokens of a block and head (the format and layout stand in ``qwen36_hip.h``).  A run's scale fits the values that the call
    writes to it; a call that goes on with a run never makes its scale smaller, and where it grows, rounds the codes of the
    tokens before to it; values behind the call's last token of a run are lost.  ``slots`` ``(tokens,)`` hold ``block id * block_size + position % block_size``
    (:func:`paged_kv_plan`); those outside the pool, such as -1, are skipped.  They have to be distinct, and the tokens of a
    run have to follow one another, with none but skipped ones between them, as a plan's do.
    """
    _tiles_append("paged_kv8_append", _kv8_descriptor, key, value, key_pool, value_pool, slots, block_size)


def paged_kv8_gather(key_pool: torch.Tensor, value_pool: torch.Tensor, block_tables: torch.Tensor, valid: int, block_size: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Dense ``(B, H_kv, valid, D)`` bf16 K/V of an 8-bit pool in logical order (:func:`paged_kv_gather`'s counterpart).

    Every value the cache holds is exact in bf16.  Tokens whose block id is outside the pool, or past the table, are
    zeros; a value stored from an infinity or a NaN reads as NaN.
    """
    return _tiles_gather("paged_kv8_gather", _kv8_descriptor, key_pool, value_pool, block_tables, valid, block_size)


def paged_attention_decode_kv8(
    query: torch.Tensor,
    block_tables: torch.Tensor,
    key_pool: torch.Tensor,
    value_pool: torch.Tensor,
    sequence_lengths: torch.Tensor,
    block_size: int,
    *,
    gate: torch.Tensor | None = None,
    scale: float | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``paged_attention_decode_batched`` over an 8-bit pool: one token per row, ``query`` ``(B, H, 1, D)`` bf16.

    ``gate`` ``(B, H*D)`` or ``(B, H, D)`` bf16 logits (a view of ``q_proj`` is read in place) give ``out *
    sigmoid(gate)``.  Rows of length <= 0, and rows that see only blocks outside the pool, give zeros.  Returns
    ``(B, H, 1, D)`` bf16, in ``out`` where it is given.
    """
    return _tiles_decode("paged_attention_decode_kv8", _kv8_descriptor, query, block_tables, key_pool, value_pool, sequence_lengths, block_size, gate, scale, out)


def paged_attention_prefill_kv8(
    query: torch.Tensor,
    cu_seqlens: torch.Tensor,
    prefix_lens: torch.Tensor,
    key_pool: torch.Tensor,
    value_pool: torch.Tensor,
    block_tables: torch.Tensor,
    block_size: int,
    *,
    max_new: int,
    gate: torch.Tensor | None = None,
    scale: float | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """:func:`paged_attention_prefill` over an 8-bit pool: causal attention of packed new tokens.

    ``query`` ``(tokens, H, D)`` bf16; the new tokens' K/V are in the pool already, so a new token sees itself and
    its neighbours in 8 bits, as every later step will.  ``max_new`` is at least the longest row of ``cu_seqlens``
    (tokens past it are not computed).  Returns ``(tokens, H, D)`` bf16, in ``out`` where it is given; rows past the
    last sequence are not written.
    """
    return _tiles_prefill("paged_attention_prefill_kv8", _kv8_descriptor, query, cu_seqlens, prefix_lens, key_pool, value_pool, block_tables, block_size, max_new, gate, scale, out)


class PagedCopy(NamedTuple):
    """Pages to be copied (:func:`paged_kv_copy`): int32 ``sources`` and ``targets``, -1 where there is none."""

    sources: torch.Tensor
    targets: torch.Tensor


def _books(
    device: torch.device, block_tables: torch.Tensor, lengths: torch.Tensor | None, free_list: torch.Tensor, free_state: torch.Tensor, references: torch.Tensor, status: torch.Tensor,
) -> tuple[int, int]:
    """Checks the books of a pool; their rows and the table's width."""
    i32 = torch.int32
    shape = block_tables.shape
    if (
        device.type == "cuda" and free_list.device == free_state.device == references.device == status.device == device
        and block_tables.dtype is i32 and len(shape) == 2 and block_tables.stride(1) == 1 and shape[0] > 0 and shape[1] > 0
        and (lengths is None or (lengths.device == device and lengths.dtype is i32 and lengths.shape == shape[:1] and lengths.is_contiguous()))
        and free_list.dtype is i32 and free_list.dim() == 1 and free_list.is_contiguous() and free_state.dtype is i32 and free_state.shape == (2,) and free_state.is_contiguous()
        and references.dtype is i32 and references.shape == free_list.shape and references.is_contiguous() and status.dtype is i32 and status.numel() >= 1
    ):
        return shape
    _same_device(device, block_tables=block_tables, lengths=block_tables if lengths is None else lengths, free_list=free_list, free_state=free_state, references=references, status=status)
    _require(block_tables.dtype is i32 and len(shape) == 2 and block_tables.stride(1) == 1, "block_tables must be int32 [rows, max_blocks] with contiguous rows")
    _require(shape[0] > 0 and shape[1] > 0, "block_tables must have shape [rows, max_blocks]")
    _require(lengths is None or (lengths.dtype is i32 and lengths.shape == shape[:1] and lengths.is_contiguous()), "lengths must be a contiguous int32 [rows] tensor")
    _require(free_list.dtype is i32 and free_list.dim() == 1 and free_list.is_contiguous(), "free_list must be a contiguous int32 vector")
    _require(free_state.dtype is i32 and free_state.shape == (2,) and free_state.is_contiguous(), "free_state must be int32 [head, count]")
    _require(references.dtype is i32 and references.shape == free_list.shape and references.is_contiguous(), "references must be a contiguous int32 tensor with an entry for each block")
    raise RuntimeError("status must be an int32 tensor")


def _row_list(rows: torch.Tensor, name: str, device: torch.device) -> torch.Tensor:
    if rows.device != device:
        _require_cuda(rows, name, device)
    _index_dtype(rows, name)
    _require(rows.dim() == 1, f"{name} must be a vector of table rows")
    return rows.contiguous()


def paged_kv_fork(
    block_tables: torch.Tensor, lengths: torch.Tensor, source_rows: torch.Tensor, target_rows: torch.Tensor, free_list: torch.Tensor, free_state: torch.Tensor,
    references: torch.Tensor, status: torch.Tensor, block_size: int,
) -> PagedCopy:
    """Makes each row ``target_rows[i]`` a copy of row ``source_rows[i]`` on the device, without copying what is full.

    The new row shares the source's full blocks (``references`` ``(blocks,)`` int32 counts a block's holders beyond its first)
    and takes the next block of the ascending ``free_list`` for a partly filled last one: the returned pages are to be copied in
    every layer's pools (:func:`paged_kv_copy`) before either row grows.  Target rows have to be empty (length 0), distinct
    and no sources; a source of -1 is no fork; at most 1024 a call.  Tables, lengths and ``free_state`` are those of
    :func:`paged_kv_plan`.  ``status`` becomes 0, or 1 (pool exhausted), 3 (corrupt free state), 4 (a length that the table does
    not hold), 6 (rows out of range, targets that are not empty or not distinct): then nothing is changed and no page is to be
    copied; as for the other calls on pages it is a tensor other than the plan's, whose refusal a success would overwrite.
    Nothing is read back, so the call can be captured in a HIP graph.
    """
    lib = L.load_library()
    device = block_tables.device
    rows, max_blocks = _books(device, block_tables, lengths, free_list, free_state, references, status)
    source, target = _row_list(source_rows, "source_rows", device), _row_list(target_rows, "target_rows", device)
    _require(source.shape == target.shape and source.dtype is target.dtype, "source_rows and target_rows must be alike")
    n = source.numel()
    pages = lengths.new_empty((2, n))
    code = _launch(
        device, lib.qa_paged_kv_fork, block_tables.data_ptr(), block_tables.stride(0), max_blocks, lengths.data_ptr(), rows, source.data_ptr(), target.data_ptr(), _code(source), n,
        int(block_size), free_list.data_ptr(), free_list.numel(), free_state.data_ptr(), references.data_ptr(), status.data_ptr(), pages.data_ptr(), pages.data_ptr() + 4 * n,
    )
    L.check(lib, code, "paged_kv_fork")
    return PagedCopy(*pages.unbind())


def paged_kv_release(
    block_tables: torch.Tensor, lengths: torch.Tensor, release_rows: torch.Tensor, free_list: torch.Tensor, free_state: torch.Tensor, references: torch.Tensor,
    status: torch.Tensor,
) -> None:
    """Frees the blocks of ``release_rows`` on the device and empties the rows.

    A block that other rows hold too (:func:`paged_kv_fork`) loses a holder, the others go back to ``free_list``, which is then
    ascending from its front.  Rows out of range are skipped, a row named twice is freed once.  ``status`` becomes 0, or 3
    (corrupt free state: nothing is changed).  The device form of ``DeviceBlockAllocator.release``: nothing is read back.
    """
    lib = L.load_library()
    device = block_tables.device
    rows, max_blocks = _books(device, block_tables, lengths, free_list, free_state, references, status)
    which = _row_list(release_rows, "release_rows", device)
    nbytes = lib.qa_paged_kv_release_workspace(free_list.numel(), which.numel(), max_blocks)
    ws = torch.zeros(nbytes // 4, dtype=torch.int32, device=device) if nbytes else None
    code = _launch(
        device, lib.qa_paged_kv_release, block_tables.data_ptr(), block_tables.stride(0), max_blocks, lengths.data_ptr(), rows, which.data_ptr(), _code(which), which.numel(),
        free_list.data_ptr(), free_list.numel(), free_state.data_ptr(), references.data_ptr(), status.data_ptr(), _ptr(ws), nbytes,
    )
    L.check(lib, code, "paged_kv_release")


def paged_kv_compact(
    block_tables: torch.Tensor, free_list: torch.Tensor, free_state: torch.Tensor, references: torch.Tensor, status: torch.Tensor, *, max_moves: int,
) -> PagedCopy:
    """Moves the blocks of the tables to the pool's lowest ids, at most ``max_moves`` of them, on the device.

    The largest id that the tables hold takes the lowest free one, and so on as long as that is lower: tables, ``references``
    and ``free_list`` are as after the moves, and the returned pages ``(max_moves,)`` are to be copied in every layer's pools
    (:func:`paged_kv_copy`).  Blocks that are neither free nor in these tables (another batch's, a host cache's) stay.
    ``status`` becomes 0, or 3 (corrupt free state: nothing is changed).  Nothing is read back.
    """
    lib = L.load_library()
    device = block_tables.device
    rows, max_blocks = _books(device, block_tables, None, free_list, free_state, references, status)
    max_moves = int(max_moves)
    _require(max_moves >= 0, "max_moves must be non-negative")
    pages = block_tables.new_empty((2, max_moves))
    nbytes = lib.qa_paged_kv_compact_workspace(free_list.numel(), rows, max_blocks, max_moves)
    ws = torch.zeros(nbytes // 4, dtype=torch.int32, device=device) if nbytes else None
    code = _launch(
        device, lib.qa_paged_kv_compact, block_tables.data_ptr(), block_tables.stride(0), max_blocks, rows, free_list.data_ptr(), free_list.numel(), free_state.data_ptr(),
        references.data_ptr(), status.data_ptr(), max_moves, pages.data_ptr(), pages.data_ptr() + 4 * max_moves, _ptr(ws), nbytes,
    )
    L.check(lib, code, "paged_kv_compact")
    return PagedCopy(*pages.unbind())


class PagePools:
    """Pools whose pages can be copied, checked once (:func:`page_pools`)."""

    __slots__ = ("device", "bases", "strides", "sizes", "counts", "tensors")


def page_pools(pools: Sequence[torch.Tensor]) -> PagePools:
    """The pools as :func:`paged_kv_copy` takes them, or its ``RuntimeError`` for what it cannot copy: a caller whose books
    change before the copy asks first."""
    pools = list(pools)
    n = len(pools)
    _require(n > 0, "pools must name at least one tensor")
    first = pools[0]
    device, shape, dtype = first.device, first.shape, first.dtype
    if device.type != "cuda":
        _require_cuda(first, "pools")
    described = PagePools()
    described.tensors, described.device = pools, device
    index = first.get_device()
    addresses, bits = [], 0
    alike = len(shape) > 1 and shape[0] > 0
    for pool in pools:
        at = pool.data_ptr()
        addresses.append(at)
        bits |= at
        if alike and not (pool.is_contiguous() and pool.shape == shape and pool.dtype is dtype and pool.get_device() == index):
            alike = False
    if alike:
        size = first.numel() // shape[0] * first.element_size()
        bits |= size
        described.sizes = described.strides = array("q", (size,)) * n
        described.counts = array("q", (shape[0],)) * n
        _require(0 not in addresses, "pools must have memory")
    else:
        for pool in pools:
            if pool.device != device:
                _require_cuda(pool, "pools", device)
            _require(pool.dim() > 1 and (pool.numel() == 0 or pool[0].is_contiguous()), "a pool's pages must be contiguous along its first axis")
        sizes = [math.prod(pool.shape[1:]) * pool.element_size() for pool in pools]
        strides = [pool.stride(0) * pool.element_size() for pool in pools]
        for pool, at, size, stride in zip(pools, addresses, sizes, strides):
            _require(at != 0 or pool.shape[0] == 0, "pools must have memory")
            _require(stride >= size or pool.shape[0] <= 1, "pages of a pool overlap")
            bits |= size | stride
        described.sizes, described.strides = array("q", sizes), array("q", strides)
        described.counts = array("q", [pool.shape[0] for pool in pools])
    _require(bits & 3 == 0, "pages of pools must be of 4-byte units")
    described.bases = array("Q", addresses)
    return described


def paged_kv_copy(pools: Sequence[torch.Tensor] | PagePools, sources: torch.Tensor, targets: torch.Tensor) -> None:
    """Copies page ``sources[i]`` to page ``targets[i]`` of every pool, in place.

    A pool is any tensor whose first axis counts pages of contiguous elements: ``(P, H_kv, bs, D)``, 4- or 8-bit tiles, states of
    a ``LinearStatePool``; a page's size and stride are multiples of 4 bytes.  Pairs with an id outside a pool, such as -1,
    are skipped there.  Targets have to be distinct, and none may be a source, as the pages of :func:`paged_kv_fork` and
    :func:`paged_kv_compact` are.
    """
    lib = L.load_library()
    if not isinstance(pools, PagePools):
        pools = page_pools(pools)
    device = pools.device
    if not (sources.device == targets.device == device):
        _same_device(device, sources=sources, targets=targets)
    _index_dtype(sources, "sources")
    _require(sources.dtype is targets.dtype and sources.dim() == 1 and sources.shape == targets.shape, "sources and targets must be vectors of page ids, alike")
    s, t = sources.contiguous(), targets.contiguous()
    code = _launch(
        device, lib.qa_paged_kv_copy, pools.bases.buffer_info()[0], pools.strides.buffer_info()[0], pools.sizes.buffer_info()[0], pools.counts.buffer_info()[0],
        len(pools.tensors), s.data_ptr(), t.data_ptr(), _code(s), s.numel(),
    )
    L.check(lib, code, "paged_kv_copy")


def mrope_axes(sections: Sequence[int], interleaved: bool) -> list[int]:
    """The position axis of each of the ``sum(sections)`` frequencies.

    Section ``a`` counts the frequencies of axis ``a``.  In order: the first ``sections[0]`` are axis 0's, the next
    axis 1's, and so on.  Interleaved: with ``n`` axes, axis ``a > 0`` has frequencies ``a, a + n, ..`` below
    ``n * sections[a]``, and axis 0 all others.
    """
    sections = [int(s) for s in sections]
    _require(1 <= len(sections) <= 4 and min(sections) >= 0 and sum(sections) > 0, "sections must be 1 to 4 counts of frequencies")
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    axes = [0] * sum(sections)
    for a in range(1, len(sections)):
        for j in range(a, min(len(sections) * sections[a], len(axes)), len(sections)):
            axes[j] = a
    return axes


_MROPE: dict[tuple[Any, ...], tuple[torch.Tensor, torch.Tensor]] = {}


def _mrope_tables(sections: tuple[int, ...], interleaved: bool, rope_theta: float, device: torch.device) -> tuple[torch.Tensor, torch.Tensor]:
    """The frequencies ``theta^(-j / half) / (2 pi)`` as fractions of 2^64 (int64) and their axes (uint8), cached: they
    depend on the model's configuration alone."""
    key = (sections, interleaved, rope_theta, device)
    cached = _MROPE.get(key)
    if cached is None:
        # made by a copy from the host that waits: not while a graph records
        _require(not torch.cuda.is_current_stream_capturing(), "the first prologue with these sections and rope_theta must run outside a graph capture")
        _require(rope_theta >= 1.0, "rope_theta must be at least 1")
        axes = mrope_axes(sections, interleaved)
        turns = [round(math.ldexp(rope_theta ** (-j / len(axes)) / (2 * math.pi), 64)) for j in range(len(axes))]
        cached = (torch.tensor(turns, dtype=torch.int64, device=device), torch.tensor(axes, dtype=torch.uint8, device=device))
        _MROPE[key] = cached
    return cached


def qk_norm_mrope_kv_append(
    q_proj: torch.Tensor,
    k_proj: torch.Tensor,
    v_proj: torch.Tensor,
    q_norm_weight: torch.Tensor,
    k_norm_weight: torch.Tensor,
    positions: torch.Tensor,
    sections: Sequence[int],
    key_pool: torch.Tensor,
    value_pool: torch.Tensor,
    slots: torch.Tensor,
    block_size: int,
    *,
    eps: float,
    rope_theta: float,
    interleaved: bool = False,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Prologue of a full-attention layer with rotary positions of several axes, in one launch.

    :func:`qk_norm_rope_kv_append` for tokens that have a time, a row and a column (pictures, video) rather than one
    position: ``positions`` ``(axes, tokens)`` (or ``(tokens,)``), ``sections`` and ``interleaved`` say which axis
    turns which frequency (:func:`mrope_axes`); the first ``2 * sum(sections)`` dims of a head are rotated, in pairs
    ``(j, j + sum(sections))`` by ``positions[axis(j)] * rope_theta^(-j / sum(sections))``.  fp32 throughout, rounded
    to bf16 once; angles are exact at any position.  ``sum(sections)`` is a multiple of ``D / 64``.

    ``q_proj`` ``(tokens, H, 2D)`` (query and gate halves) or ``(tokens, H, D)``, ``k_proj``/``v_proj`` ``(tokens,
    H_kv, D)``, bf16, rows aligned to ``D / 64`` elements.  Flat in the last two dims, ``q_proj`` is the form with the
    gate, ``(tokens, H*2D)``.  k and v go to ``slots`` (:func:`paged_kv_plan`; those outside the pool are skipped, the
    others have to be distinct) of a bf16 pool ``(P, H_kv, bs, D)`` or a 4-bit one ``(P, H_kv, kv4_tile_bytes(D, bs))``;
    the latter then holds what :func:`paged_kv4_append` makes of the bf16 k and v.  Returns
    ``(query (tokens, H, D) bf16, gate (tokens, H, D) view of q_proj or None)``.
    """
    lib = L.load_library()
    device = q_proj.device
    if device.type != "cuda" or not (k_proj.device == v_proj.device == q_norm_weight.device == k_norm_weight.device == positions.device == slots.device == key_pool.device == device):
        _same_device(device, q_proj=q_proj, k_proj=k_proj, v_proj=v_proj, q_norm_weight=q_norm_weight, k_norm_weight=k_norm_weight, positions=positions, key_pool=key_pool,
                     value_pool=value_pool, slots=slots)
    bf16 = torch.bfloat16
    if key_pool.dtype is torch.uint8:
        desc, head_dim = _kv4_descriptor(key_pool, value_pool, block_size, device)
    else:
        _require_cuda(value_pool, "value_pool", device)
        _require(key_pool.dtype is bf16 and key_pool.dim() == 4 and key_pool.shape[2] == block_size, "the pool must be bfloat16 (blocks, kv_heads, block_size, head_dim) or 4-bit")
        desc, head_dim = _pool_descriptor(key_pool, value_pool, "shared"), key_pool.shape[3]
    kv_heads = desc.kv_heads
    q_shape = q_proj.shape
    tokens = q_shape[0]
    k3 = k_proj.view(tokens, kv_heads, head_dim) if k_proj.dim() == 2 else k_proj
    v3 = v_proj.view(tokens, kv_heads, head_dim) if v_proj.dim() == 2 else v_proj
    q3 = q_proj
    if len(q_shape) == 2 and q_shape[1] % (2 * head_dim) == 0:
        q3 = q_proj.view(tokens, q_shape[1] // (2 * head_dim), 2 * head_dim)
        q_shape = q3.shape
    _require(len(q_shape) == 3 and q_shape[2] in (head_dim, 2 * head_dim), "q_proj must be (tokens, heads, head_dim or 2*head_dim) or (tokens, heads*2*head_dim)")
    heads = q_shape[1]
    _require(k3.shape == (tokens, kv_heads, head_dim) and v3.shape == k3.shape, "k_proj/v_proj must be (tokens, kv_heads, head_dim)")
    q_st, q_sh, q_sd = q3.stride()
    k_st, k_sh, k_sd = k3.stride()
    v_st, v_sh, v_sd = v3.stride()
    if not (q3.dtype is bf16 and k3.dtype is bf16 and v3.dtype is bf16 and q_sd == k_sd == v_sd == 1):
        raise RuntimeError("q_proj, k_proj and v_proj must be bfloat16 with a contiguous last dimension")
    _float_dtype(q_norm_weight, "q_norm_weight")
    _require(q_norm_weight.dtype is k_norm_weight.dtype and q_norm_weight.shape == (head_dim,) and k_norm_weight.shape == (head_dim,),
             "norm weights must be (head_dim,) of one dtype")
    _index_dtype(positions, "positions")
    _index_dtype(slots, "slots")
    sections = tuple(sections)
    pos = positions.unsqueeze(0) if positions.dim() == 1 else positions
    _require(pos.shape == (len(sections), tokens), "positions must be (axes, tokens), one axis per section")
    _require(slots.shape == (tokens,), "slots must have one entry per token")
    freq, axis = _mrope_tables(sections, bool(interleaved), float(rope_theta), device)
    pos_stride, pos_unit = pos.stride()
    if pos_unit != 1:
        pos = pos.contiguous()
        pos_stride = tokens
    s, qw, kw = slots.contiguous(), q_norm_weight.contiguous(), k_norm_weight.contiguous()
    query = torch.empty((tokens, heads, head_dim), dtype=bf16, device=device)
    code = _launch(
        device, lib.qa_qk_norm_mrope_append, q3.data_ptr(), q_st, q_sh, k3.data_ptr(), k_st, k_sh, v3.data_ptr(), v_st, v_sh, qw.data_ptr(), kw.data_ptr(), _code(qw),
        float(eps), freq.data_ptr(), axis.data_ptr(), 2 * axis.numel(), pos.data_ptr(), _code(pos), pos_stride, len(sections), tokens, heads, head_dim, ctypes.byref(desc),
        s.data_ptr(), _code(s), int(block_size), query.data_ptr(),
    )
    L.check(lib, code, "qk_norm_mrope_kv_append")
    return query, q3.narrow(2, head_dim, head_dim) if q_shape[2] == 2 * head_dim else None
