"""What the entry points of the 4-bit cache refuse, on the host, before any launch."""

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


def _desc(**changes) -> L.PagedKV:
    desc = L.PagedKV(1 << 20, 1 << 20, None, None, None, 8, 0, 2 * 2176, 2176, 0, 2, L.QA_KV4)
    for name, value in changes.items():
        setattr(desc, name, value)
    return desc


def _append(lib, desc=None, **changes) -> int:
    a = dict(key=SOME, value=SOME, dtype=L.QA_BF16, kt=512, kh=256, vt=512, vh=256, tokens=3, dim=256, slots=SOME, slots_dtype=L.QA_I64, block=16)
    a.update(changes)
    return lib.qa_paged_kv4_append(a["key"], a["value"], a["dtype"], a["kt"], a["kh"], a["vt"], a["vh"], a["tokens"], a["dim"], ctypes.byref(desc or _desc()), a["slots"],
                                   a["slots_dtype"], a["block"], P(0))


BAD_POOLS = [
    (dict(dtype=L.QA_BF16), "must be a 4-bit pool"), (dict(key=None), "one shared pool"), (dict(row_key_ptrs=1 << 20), "one shared pool"),
    (dict(kv_heads=0), "kv_heads"), (dict(num_blocks=-1), "kv_heads"), (dict(num_blocks=1 << 31), "fit int32"), (dict(stride_head=2160), "smaller than a tile"),
    (dict(stride_block=2160), "smaller than a tile"), (dict(key=(1 << 20) + 8), "16-byte aligned"), (dict(stride_head=2184), "16-byte aligned"),
]


@pytest.mark.parametrize("changes,message", BAD_POOLS)
def test_every_entry_refuses_a_bad_pool(changes, message) -> None:
    lib = _lib()
    desc = _desc(**changes)
    calls = {
        "append": _append(lib, desc),
    }
    assert calls["append"] == 1 and message in L.last_error(lib)
    assert lib.qa_paged_kv4_gather(ctypes.byref(desc), 256, 1, SOME, L.QA_I32, 4, 4, 16, 16, SOME, SOME, P(0)) == 1
    assert message in L.last_error(lib)
    assert lib.qa_paged_attention_decode_kv4(SOME, L.QA_BF16, 4096, 256, 1, 16, 256, ctypes.byref(desc), SOME, L.QA_I32, 4, 4, SOME, L.QA_I32, 16, 0.0, P(0), 0, 0, SOME, SOME,
                                             1 << 30, P(0)) == 1
    assert message in L.last_error(lib)
    assert lib.qa_paged_attention_prefill_kv4(SOME, L.QA_BF16, 4096, 256, 3, SOME, SOME, L.QA_I32, 1, 3, 16, 256, ctypes.byref(desc), SOME, L.QA_I32, 4, 4, 16, 0.0, P(0), 0, 0,
                                              SOME, SOME, 1 << 30, P(0)) == 1
    assert message in L.last_error(lib)


@pytest.mark.parametrize("changes,message", [
    (dict(dtype=L.QA_F16), "float32 or bfloat16"), (dict(dim=64), "head_dim"), (dict(dim=192), "head_dim"), (dict(block=8), "block_size"), (dict(block=48), "block_size"),
    (dict(block=2048), "block_size"), (dict(slots_dtype=L.QA_F32), "int32 or int64"), (dict(key=P(0)), "non-null"), (dict(slots=P(0)), "non-null"), (dict(kt=516), "aligned"),
    (dict(key=P((1 << 20) + 8)), "aligned"), (dict(tokens=-1), "out of range"),
])
def test_append_refuses(changes, message) -> None:
    lib = _lib()
    assert _append(lib, **changes) == 1
    assert message in L.last_error(lib)


def test_nothing_to_do_is_no_error() -> None:
    lib = _lib()
    assert _append(lib, tokens=0, key=P(0), value=P(0), slots=P(0)) == 0
    assert lib.qa_paged_kv4_gather(ctypes.byref(_desc()), 256, 1, SOME, L.QA_I32, 4, 4, 0, 16, P(0), P(0), P(0)) == 0


def _decode(lib, **changes) -> int:
    a = dict(q=SOME, dtype=L.QA_BF16, qb=4096, qh=256, batch=1, heads=16, dim=256, tables=SOME, tdtype=L.QA_I32, stride=4, width=4, lens=SOME, ldtype=L.QA_I32, block=16, gate=P(0),
             gb=0, gh=0, out=SOME, ws=SOME, wsb=1 << 30)
    a.update(changes)
    return lib.qa_paged_attention_decode_kv4(a["q"], a["dtype"], a["qb"], a["qh"], a["batch"], a["heads"], a["dim"], ctypes.byref(_desc()), a["tables"], a["tdtype"], a["stride"],
                                             a["width"], a["lens"], a["ldtype"], a["block"], 0.0, a["gate"], a["gb"], a["gh"], a["out"], a["ws"], a["wsb"], P(0))


BAD_ATTENTION = [
    (dict(dtype=L.QA_F32), "must be bfloat16"), (dict(tdtype=L.QA_F32), "int32/int64"), (dict(heads=15), "multiple of KV heads"), (dict(heads=34), "larger than 16"),
    (dict(heads=0), "multiple of KV heads"), (dict(width=0), "at least one entry"), (dict(qb=1 << 32), "strides"), (dict(gate=SOME, gb=1 << 33), "strides"), (dict(qh=-256), "strides"), (dict(qb=4100), "16-byte aligned"), (dict(q=P((1 << 20) + 8)), "16-byte aligned"),
    (dict(gate=P((1 << 20) + 2)), "8-byte aligned"), (dict(gate=SOME, gb=2), "8-byte aligned"), (dict(q=P(0)), "non-null"), (dict(out=P(0)), "non-null"), (dict(tables=P(0)), "non-null"),
    (dict(batch=-1), "out of range"),
]


@pytest.mark.parametrize("changes,message", BAD_ATTENTION + [(dict(lens=P(0)), "device array"), (dict(ldtype=L.QA_F32), "int32/int64")])
def test_decode_refuses(changes, message) -> None:
    lib = _lib()
    assert _decode(lib, **changes) == 1
    assert message in L.last_error(lib)


@pytest.mark.parametrize("changes,message", BAD_ATTENTION + [(dict(cu=P(0)), "non-null"), (dict(total=-1), "out of range"), (dict(max_new=-1), "out of range"),
                                                             (dict(width=4000, wsb=4), "workspace too small")])
def test_prefill_refuses(changes, message) -> None:
    lib = _lib()
    a = dict(q=SOME, dtype=L.QA_BF16, qb=4096, qh=256, total=3, cu=SOME, prefix=SOME, batch=1, max_new=3, heads=16, dim=256, tables=SOME, tdtype=L.QA_I32, stride=4, width=4,
             block=16, gate=P(0), gb=0, out=SOME)
    a.update(changes)
    assert lib.qa_paged_attention_prefill_kv4(a["q"], a["dtype"], a["qb"], a["qh"], a["total"], a["cu"], a["prefix"], L.QA_I32, a["batch"], a["max_new"], a["heads"], a["dim"],
                                              ctypes.byref(_desc()), a["tables"], a["tdtype"], a["stride"], a["width"], a["block"], 0.0, a["gate"], a["gb"], 0, a["out"],
                                              SOME, a.get("wsb", 1 << 30), P(0)) == 1
    assert message in L.last_error(lib)


@pytest.mark.parametrize("changes,message", [
    (dict(batch=0), "batch"), (dict(tables=P(0)), "non-null"), (dict(counts_dtype=L.QA_F32, counts=SOME), "counts"), (dict(scalar=-1), "non-negative"), (dict(block=0), "block_size"),
    (dict(stride=3), "overlap"), (dict(capacity=0), "capacity"), (dict(max_tokens=-1), "max_tokens"), (dict(positions=P(0)), "non-null"), (dict(wsb=4), "workspace too small"),
    (dict(per_row=-1), "entries a row"), (dict(per_row=3), "max_tokens must be 6"),
])
def test_plan_refuses(changes, message) -> None:
    lib = _lib()
    a = dict(tables=SOME, stride=4, width=4, counts=P(0), counts_dtype=L.QA_I32, scalar=1, batch=2, block=16, capacity=8, max_tokens=4, positions=SOME, wsb=8, per_row=0)
    a.update(changes)
    assert lib.qa_paged_kv_plan(a["tables"], a["stride"], a["width"], SOME, a["counts"], a["counts_dtype"], a["scalar"], a["batch"], a["block"], SOME, a["capacity"], SOME, SOME,
                                a["max_tokens"], a["per_row"], SOME, SOME, a["positions"], SOME, SOME, a["wsb"], P(0)) == 1
    assert message in L.last_error(lib)


@pytest.mark.parametrize("changes,message", [
    (dict(dtype=L.QA_F32), "bfloat16 or 4-bit"), (dict(dim=96), "head_dim"), (dict(wdtype=L.QA_F16), "norm weights"), (dict(rd=0), "rotary_dim"), (dict(rd=6), "rotary_dim"),
    (dict(rd=264), "rotary_dim"), (dict(axes=0), "axes"), (dict(axes=5), "axes"), (dict(heads=15), "multiple of KV heads"), (dict(eps=-1.0), "eps"), (dict(tokens=-1), "out of range"),
    (dict(q=P(0)), "non-null"), (dict(qt=4098), "aligned"), (dict(k=P((1 << 20) + 4)), "aligned"),
])
def test_mrope_prologue_refuses(changes, message) -> None:
    lib = _lib()
    a = dict(q=SOME, qt=8192, k=SOME, wdtype=L.QA_BF16, eps=1e-6, rd=64, axes=3, tokens=5, heads=16, dim=256, dtype=L.QA_KV4)
    a.update(changes)
    desc = _desc(dtype=a["dtype"])
    assert lib.qa_qk_norm_mrope_append(a["q"], a["qt"], 512, a["k"], 512, 256, SOME, 512, 256, SOME, SOME, a["wdtype"], a["eps"], SOME, SOME, a["rd"], SOME, L.QA_I32, 5, a["axes"],
                                       a["tokens"], a["heads"], a["dim"], ctypes.byref(desc), SOME, L.QA_I64, 16, SOME, P(0)) == 1
    assert message in L.last_error(lib)


def test_cpu_tensors_and_bad_geometry_raise() -> None:
    x = torch.zeros(1)
    for call in (
        lambda: hip_ops.paged_kv_plan(x, x, 1, x, x, x, 16, max_tokens=1),
        lambda: hip_ops.paged_kv4_append(x, x, x, x, x, 16),
        lambda: hip_ops.paged_kv4_gather(x, x, x, 1, 16),
        lambda: hip_ops.paged_attention_decode_kv4(x, x, x, x, x, 16),
        lambda: hip_ops.paged_attention_prefill_kv4(x, x, x, x, x, x, 16, max_new=1),
        lambda: hip_ops.qk_norm_mrope_kv_append(x, x, x, x, x, x, (1,), x, x, x, 16, eps=1e-6, rope_theta=1e4),
    ):
        with pytest.raises(RuntimeError, match="must be CUDA"):
            call()
    for dim, block in ((64, 16), (256, 8), (256, 24), (256, 2048)):
        with pytest.raises(RuntimeError):
            hip_ops.kv4_tile_bytes(dim, block)
    for sections in ((), (0, 0), (1, 1, 1, 1, 1), (3, -1)):
        with pytest.raises(RuntimeError):
            hip_ops.mrope_axes(sections, False)
