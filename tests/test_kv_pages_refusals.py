"""What the entry points of a cache's pages refuse, on the host, before any launch."""

from __future__ import annotations

import ctypes

import pytest
import torch

import hip_loader as L
import hip_ops

P = ctypes.c_void_p
SOME = P(1 << 20)  # an aligned address that no refused call follows


def _lib():
    if not L.LIBRARY_PATH.exists():
        pytest.fail(f"{L.LIBRARY_PATH} is not built; run __graft_entry__.build()")
    return L.load_library()


BOOKS = dict(tables=SOME, stride=4, width=4, lengths=SOME, rows=3, which=SOME, dtype=L.QA_I32, n=2, free=SOME, capacity=8, state=SOME, references=SOME, status=SOME, ws=SOME, wsb=1 << 20)
BAD_BOOKS = [
    (dict(tables=P(0)), "non-null"), (dict(free=P(0)), "non-null"), (dict(state=P(0)), "non-null"), (dict(references=P(0)), "non-null"), (dict(status=P(0)), "non-null"),
    (dict(rows=0), "rows"), (dict(rows=65534), "rows"), (dict(width=0), "at least one entry"), (dict(stride=3), "overlap"), (dict(capacity=0), "capacity"), (dict(capacity=1 << 31), "capacity"),
]


def _fork(lib, **changes) -> int:
    a = dict(BOOKS, target=SOME, block=16, sources=SOME, targets=SOME)
    a.update(changes)
    return lib.qa_paged_kv_fork(a["tables"], a["stride"], a["width"], a["lengths"], a["rows"], a["which"], a["target"], a["dtype"], a["n"], a["block"], a["free"], a["capacity"],
                                a["state"], a["references"], a["status"], a["sources"], a["targets"], P(0))


def _release(lib, **changes) -> int:
    a = dict(BOOKS)
    a.update(changes)
    return lib.qa_paged_kv_release(a["tables"], a["stride"], a["width"], a["lengths"], a["rows"], a["which"], a["dtype"], a["n"], a["free"], a["capacity"], a["state"], a["references"],
                                   a["status"], a["ws"], a["wsb"], P(0))


def _compact(lib, **changes) -> int:
    a = dict(BOOKS, moves=5, sources=SOME, targets=SOME)
    a.update(changes)
    return lib.qa_paged_kv_compact(a["tables"], a["stride"], a["width"], a["rows"], a["free"], a["capacity"], a["state"], a["references"], a["status"], a["moves"], a["sources"],
                                   a["targets"], a["ws"], a["wsb"], P(0))


@pytest.mark.parametrize("changes,message", BAD_BOOKS + [
    (dict(dtype=L.QA_F32), "int32 or int64"), (dict(n=-1), "forks"), (dict(n=1025), "forks"), (dict(block=0), "block_size"), (dict(block=65537), "block_size"), (dict(lengths=P(0)), "non-null"),
    (dict(which=P(0)), "non-null"), (dict(target=P(0)), "non-null"), (dict(sources=P(0)), "non-null"), (dict(targets=P(0)), "non-null"),
])
def test_fork_refuses(changes, message) -> None:
    lib = _lib()
    assert _fork(lib, **changes) == 1
    assert message in L.last_error(lib)


@pytest.mark.parametrize("changes,message", BAD_BOOKS + [
    (dict(dtype=L.QA_F32), "int32 or int64"), (dict(n=-1), "rows a call"), (dict(n=65534), "rows a call"), (dict(lengths=P(0)), "non-null"), (dict(which=P(0)), "non-null"),
    (dict(capacity=40_000, ws=P(0)), "workspace"), (dict(capacity=40_000, wsb=5003), "workspace"), (dict(capacity=40_000, ws=P((1 << 20) + 2)), "workspace"),
    (dict(width=9000, stride=9000, ws=P(0)), "workspace"),
])
def test_release_refuses(changes, message) -> None:
    lib = _lib()
    assert _release(lib, **changes) == 1
    assert message in L.last_error(lib)


@pytest.mark.parametrize("changes,message", BAD_BOOKS + [
    (dict(moves=-1), "max_moves"), (dict(moves=1 << 31), "max_moves"), (dict(sources=P(0)), "non-null"), (dict(targets=P(0)), "non-null"),
    (dict(capacity=40_000, ws=P(0)), "workspace"), (dict(capacity=40_000, wsb=175_003), "workspace"), (dict(width=9000, stride=9000, ws=P(0)), "workspace"),
    (dict(moves=40_000, ws=P(0)), "workspace"),
])
def test_compact_refuses(changes, message) -> None:
    lib = _lib()
    assert _compact(lib, **changes) == 1
    assert message in L.last_error(lib)


def _copy(lib, base=1 << 20, stride=64, size=64, count=4, pools=1, sources=SOME, targets=SOME, dtype=L.QA_I32, n=2) -> int:
    longs = ctypes.c_int64 * 1
    return lib.qa_paged_kv_copy((ctypes.c_void_p * 1)(base), longs(stride), longs(size), longs(count), pools, sources, targets, dtype, n, P(0))


@pytest.mark.parametrize("changes,message", [
    (dict(base=None), "null"), (dict(base=(1 << 20) + 2), "4-byte units"), (dict(stride=66), "4-byte units"), (dict(size=62), "4-byte units"), (dict(stride=60), "overlap"), (dict(count=-1), "overlap"),
    (dict(size=-4), "overlap"), (dict(sources=P(0)), "non-null"), (dict(targets=P(0)), "non-null"), (dict(dtype=L.QA_F32), "int32 or int64"), (dict(n=-1), "out of range"),
    (dict(pools=-1), "out of range"),
])
def test_copy_refuses(changes, message) -> None:
    lib = _lib()
    assert _copy(lib, **changes) == 1
    assert message in L.last_error(lib)


def test_nothing_to_copy_is_no_error() -> None:
    lib = _lib()
    assert _copy(lib, n=0, sources=P(0), targets=P(0)) == 0
    assert _copy(lib, pools=0) == 0


def test_cpu_tensors_raise() -> None:
    x = torch.zeros(2, 2, dtype=torch.int32)
    for call in (
        lambda: hip_ops.paged_kv_fork(x, x[0], x[0], x[0], x[0], x[0], x[0], x[0], 16),
        lambda: hip_ops.paged_kv_release(x, x[0], x[0], x[0], x[0], x[0], x[0]),
        lambda: hip_ops.paged_kv_compact(x, x[0], x[0], x[0], x[0], max_moves=1),
        lambda: hip_ops.paged_kv_copy([x], x[0], x[0]),
    ):
        with pytest.raises(RuntimeError, match="must be CUDA"):
            call()
