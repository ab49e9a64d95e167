"""A full-attention layer over a KV cache held in 8 bits, and the pages of a cache, as cases that can be timed and checked.

* ``cache``    K/V quantised into the 8-bit cache through a slot map, and the cache's dense view
* ``decode``   one token per sequence over the 8-bit cache
* ``prefill``  a prompt, or a chunk of one, over the 8-bit cache, with the output gate
* ``pages``    ``fork``: conversations forked, their last pages copied, the parents' pages freed; ``compact``: the pages of a
  scattered cache moved to its lowest places

The 8-bit cache.  A run is 16 consecutive tokens of a block and one KV head.  It is held as 16 D E4M3 codes and a scale 2^e,
one byte e + 127.  Of the finite values written to a run in one call, e is the least integer with max |x| <= 448 2^e,
within [-117, 120]; x / 2^e goes to the nearest code, ties to the even one, and what is not finite becomes NaN.  Where the call
does not write the run's first token, e is not below what the run has, and if it is above, the codes of the tokens before the
first new one are rounded to it.  The pools are float8_e4m3fn ``(blocks, kv_heads, block_size * (D + 1))``: per block and
head, runs of 16 tokens, each first the codes, then 16 bytes, the scale's and zeros:

* keys    codes  [D/64][dim / 16 % 4][token][16 dims]
* values  codes  [D/64][token / 4][dim / 4 % 16][dim % 4][token % 4]

Pages.  ``references[id]`` counts the holders of a block beyond its first.  A fork's new row shares the full blocks of its
parent and gets a block of its own for a partly filled last one, the free list's first ids in the order of the forks.  A freed
block goes back to the list, which is then ascending from 0 and -1 behind its end.  Compaction gives the largest ids that the
tables hold the lowest free ones, the largest the lowest and so on, as long as that is a lower id.

Shapes are those of ``bench.py`` and of the tests: 16 query heads on 2 KV heads of 256 (or heads of 128) and blocks of
16 tokens, or of 32 and 64.
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

DEVICE = "cuda:0"


def listed() -> list[dict]:
    return [
        # One token for each of seven short conversations, and the cache read back dense, as a caller without paging does.
        _cache("cache_step", batch=7, new=1, prefix=427),
        # Prompts written in one go and read back.
        _cache("cache_prompt", batch=4, new=6003, prefix=0),
        # The smallest call of a chat server: four short conversations.
        _decode("decode_few", batch=4, lo=300, hi=700),
        # A full decode batch under continuous batching: 64 conversations of 1k to 32k tokens.
        _decode("decode_batch", batch=64, lo=1024, hi=32768),
        # One very long document: the sequence has to be split over the whole chip.
        _decode("decode_long", batch=1, lo=200_003, hi=200_003, heads=16, kv_heads=1, dim=128, block=64, index="int64"),
        # Fresh prompts of a few words up to a page, packed into one ragged step with nothing cached.
        _prefill("prefill_prompts", batch=5, new_lo=37, new_hi=700, prefix_lo=0, prefix_hi=0, heads=20, kv_heads=4, dim=128),
        # Chunked prefill in steady state: eight requests, 512 new tokens each, behind up to 8k cached ones.
        _prefill("prefill_chunk", batch=8, new_lo=512, new_hi=512, prefix_lo=0, prefix_hi=8192),
        # One long document's last chunk.
        _prefill("prefill_long", batch=1, new_lo=2048, new_hi=2048, prefix_lo=32_000, prefix_hi=32_000),
        # Three more answers to one question.
        _fork("fork_few", parents=1, children=3, lo=700, hi=700, layers=2),
        # A full batch of samplings: 16 prompts, eight answers each, over twelve layers of pools.
        _fork("fork_batch", parents=16, children=8, lo=100, hi=4096, layers=12),
        # A small cache after many requests have left it.
        _compact("compact_few", batch=6, lo=50, hi=900, layers=2, spare=1.5),
        # A large cache packed before its tail is given back.
        _compact("compact_batch", batch=64, lo=256, hi=8192, layers=3, spare=0.8),
    ]


def draw(rng: random.Random) -> dict:
    family = rng.choice(("cache", "cache", "decode", "decode", "prefill", "prefill", "fork", "compact"))
    block = rng.choice((16, 16, 32, 64))
    index = rng.choice(("int32", "int64"))
    if family == "cache":
        heads_dim = rng.choice(((2, 256), (2, 128), (4, 128), (1, 256)))
        new = _log_int(rng, 1, 6000)
        return _cache(None, batch=rng.randint(1, 4), new=new, prefix=rng.choice((0, _log_int(rng, 1, 6001 - new))), kv_heads=heads_dim[0], dim=heads_dim[1], block=block, index=index)
    if family == "decode":
        heads, kv_heads, dim = rng.choice(((16, 2, 256), (16, 2, 256), (8, 2, 128), (16, 1, 128), (6, 2, 256), (12, 2, 128), (16, 1, 256)))
        hi = _log_int(rng, 1, 32768)
        return _decode(None, batch=_log_int(rng, 1, 64), lo=_log_int(rng, 1, hi), hi=hi, heads=heads, kv_heads=kv_heads, dim=dim, block=block, gated=rng.random() < 0.5,
                       index=index)
    if family == "prefill":
        heads, kv_heads, dim = rng.choice(((16, 2, 256), (16, 2, 256), (8, 2, 128), (4, 4, 256), (20, 4, 128), (16, 1, 128)))
        tokens = _log_int(rng, 24, 4096)
        batch = rng.randint(1, max(1, min(8, tokens // 24)))
        new_hi = max(1, tokens // batch)
        prefix_hi = rng.choice((0, _log_int(rng, 16, 8192)))
        return _prefill(None, batch=batch, new_lo=rng.randint(max(1, new_hi // 4), new_hi), new_hi=new_hi, prefix_lo=prefix_hi // 3, prefix_hi=prefix_hi, heads=heads,
                        kv_heads=kv_heads, dim=dim, block=block, gated=rng.random() < 0.7, index=index)
    kv_heads, dim = rng.choice(((2, 256), (2, 128), (4, 128)))
    hi = _log_int(rng, 1, 4096)
    layers = rng.randint(1, 6)
    if family == "fork":
        return _fork(None, parents=_log_int(rng, 1, 16), children=rng.randint(1, 8), lo=_log_int(rng, 1, hi), hi=hi, layers=layers, kv_heads=kv_heads, dim=dim, block=block)
    return _compact(None, batch=_log_int(rng, 1, 48), lo=_log_int(rng, 1, hi), hi=hi, layers=layers, spare=round(rng.uniform(0.05, 2.0), 2), kv_heads=kv_heads, dim=dim,
                    block=block)


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _case(name, family, values) -> dict:
    case = {"family": family, **values}
    if name is not None:
        case["name"] = name
    return case


def _cache(name, *, batch, new, prefix, kv_heads=2, dim=256, block=16, index="int32"):
    return _case(name, "cache", dict(batch=batch, new=new, prefix=prefix, kv_heads=kv_heads, dim=dim, block=block, index=index))


def _decode(name, *, batch, lo, hi, heads=16, kv_heads=2, dim=256, block=16, gated=True, index="int32"):
    return _case(name, "decode", dict(batch=batch, lo=lo, hi=hi, heads=heads, kv_heads=kv_heads, dim=dim, block=block, gated=gated, index=index))


def _prefill(name, *, batch, new_lo, new_hi, prefix_lo, prefix_hi, heads=16, kv_heads=2, dim=256, block=16, gated=True, index="int32"):
    return _case(name, "prefill", dict(batch=batch, new_lo=new_lo, new_hi=new_hi, prefix_lo=prefix_lo, prefix_hi=prefix_hi, heads=heads, kv_heads=kv_heads, dim=dim,
                                       block=block, gated=gated, index=index))


def _fork(name, *, parents, children, lo, hi, layers, kv_heads=2, dim=256, block=16):
    return _case(name, "fork", dict(batch=parents, children=children, lo=lo, hi=hi, layers=layers, kv_heads=kv_heads, dim=dim, block=block))


def _compact(name, *, batch, lo, hi, layers, spare, kv_heads=2, dim=256, block=16):
    return _case(name, "compact", dict(batch=batch, lo=lo, hi=hi, layers=layers, spare=spare, kv_heads=kv_heads, dim=dim, block=block))


# --------------------------------------------------------------------------- inputs


def prepare(case: dict, seed: int):
    return {"case": case, **_INPUTS[case["family"]](case, torch.Generator(device=DEVICE).manual_seed(seed))}


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["family"]](state)


def work(case: dict) -> dict:
    return _WORK[case["family"]](case)


def exact(case: dict, seed: int):
    return _EXACT[case["family"]](prepare(case, seed))


def _randn(gen, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=gen, device=DEVICE, dtype=dtype)


def _index(case):
    return torch.int32 if case["index"] == "int32" else torch.int64


def _lengths(case: dict, what: str, lo: int, hi: int) -> list[int]:
    """Row lengths of a case: part of its shape, so they do not change with the inputs' seed."""
    rng = random.Random(f"{what} {lo} {hi} {case['batch']}")
    return [rng.randint(lo, hi) for _ in range(case["batch"])]


def _new_and_prefix(case):
    return _lengths(case, "new", case["new_lo"], case["new_hi"]), _lengths(case, "prefix", case["prefix_lo"], case["prefix_hi"])


def _int(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEVICE)


def _tables(gen, totals, block, dtype):
    """Block tables (-1 padded) over a pool with a quarter of its blocks free, blocks in random order; and the block count."""
    need = [(n + block - 1) // block for n in totals]
    blocks = math.ceil(sum(need) * 1.25) + 1
    order = torch.randperm(blocks, generator=gen, device=DEVICE)
    tables = torch.full((len(need), max(max(need), 1)), -1, dtype=dtype, device=DEVICE)
    at = 0
    for row, n in enumerate(need):
        tables[row, :n] = order[at : at + n]
        at += n
    return tables, blocks


def _channels(gen, kv_heads, dim):
    """Keys have channels far larger than the others."""
    return torch.exp(0.5 * _randn(gen, kv_heads, 1, dim, dtype=torch.float32))


def _least(top):
    """The byte of the least scale for a largest magnitude, fp32."""
    mant, expo = torch.frexp(top)  # top = mant 2^expo, mant in [0.5, 1); 448 2^(expo-9) = 0.875 2^expo
    e = torch.where(top == 0, -200, expo - 9 + (mant > 0.875))
    return e.clamp(-117, 120) + 127


def _pack(x, is_key):
    """An 8-bit pool (blocks, kv_heads, bytes) that holds x (blocks, kv_heads, block_size, dim), as bytes."""
    n, h, bs, d = x.shape
    runs = x.float().view(n, h, bs // 16, 16, d)
    byte = _least(runs.abs().amax((-1, -2)))
    codes = torch.ldexp(runs, 127 - byte[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    if is_key:
        codes = codes.view(n, h, bs // 16, 16, d // 64, 4, 16).permute(0, 1, 2, 4, 5, 3, 6)
    else:
        codes = codes.view(n, h, bs // 16, 4, 4, d // 64, 16, 4).permute(0, 1, 2, 5, 3, 6, 7, 4)
    tail = torch.zeros((n, h, bs // 16, 16), dtype=torch.uint8, device=x.device)
    tail[..., 0] = byte.to(torch.uint8)
    return torch.cat((codes.reshape(n, h, bs // 16, -1), tail), dim=-1).view(n, h, -1)


def _pools(case, gen, blocks):
    pools = []
    for is_key in (True, False):
        pool = torch.empty((blocks, case["kv_heads"], case["block"] * (case["dim"] + 1)), dtype=torch.uint8, device=DEVICE)
        scale = _channels(gen, case["kv_heads"], case["dim"]) if is_key else 1.0
        for lo in range(0, blocks, 8192):
            n = min(blocks - lo, 8192)
            pool[lo : lo + n] = _pack(_randn(gen, n, case["kv_heads"], case["block"], case["dim"], dtype=torch.float32) * scale, is_key)
        pools.append(pool.view(torch.float8_e4m3fn))
    return pools


def _cache_inputs(case, gen):
    new, prefix, kv_heads, dim, bs = case["new"], case["prefix"], case["kv_heads"], case["dim"], case["block"]
    tables, blocks = _tables(gen, [new + prefix] * case["batch"], bs, _index(case))
    keys, values = _pools(case, gen, blocks)
    at = prefix + torch.arange(new, device=DEVICE)
    slots = (tables.long()[:, at // bs] * bs + at % bs).reshape(-1)
    tokens = slots.numel()
    # some new tokens are larger than all that their run has seen
    loud = 1 + 3 * (torch.rand((tokens, 1, 1), generator=gen, device=DEVICE) < 0.3)
    return {"key": (_randn(gen, tokens, kv_heads, dim, dtype=torch.float32) * _channels(gen, kv_heads, dim).view(kv_heads, dim) * loud).bfloat16(),
            "value": (_randn(gen, tokens, kv_heads, dim, dtype=torch.float32) * loud).bfloat16(), "keys": keys, "values": values, "tables": tables, "slots": slots}


def _decode_inputs(case, gen):
    lens = _lengths(case, "context", case["lo"], case["hi"])
    tables, blocks = _tables(gen, lens, case["block"], _index(case))
    keys, values = _pools(case, gen, blocks)
    shape = (case["batch"], case["heads"], case["dim"])
    return {"query": _randn(gen, case["batch"], case["heads"], 1, case["dim"]), "gate": _randn(gen, *shape) if case["gated"] else None, "tables": tables, "keys": keys,
            "values": values, "lens": _int(lens, _index(case))}


def _prefill_inputs(case, gen):
    new, prefix = _new_and_prefix(case)
    tables, blocks = _tables(gen, [n + p for n, p in zip(new, prefix)], case["block"], _index(case))
    keys, values = _pools(case, gen, blocks)
    shape = (sum(new), case["heads"], case["dim"])
    return {"query": _randn(gen, *shape), "gate": _randn(gen, *shape) if case["gated"] else None, "tables": tables, "keys": keys, "values": values,
            "cu": _int([sum(new[:i]) for i in range(len(new) + 1)], _index(case)), "prefix": _int(prefix, _index(case)), "max_new": max(new), "new": new, "lens": prefix}


def _book(case, gen, lens, rows, blocks):
    """The books of a cache of ``rows`` rows, the first of them of ``lens`` tokens in blocks at random places: tables, lengths,
    the free list's cursor, the list and the references, side by side, so that a pass sets all of them back with one copy."""
    need = [-(-n // case["block"]) for n in lens]
    width = max(need) + 2
    book = torch.full((rows * width + rows + 2 + 2 * blocks,), -1, dtype=torch.int32, device=DEVICE)
    tables, lengths, state, free, references = book.split((rows * width, rows, 2, blocks, blocks))
    tables = tables.view(rows, width)
    order = torch.randperm(blocks, generator=gen, device=DEVICE).to(torch.int32)
    at = 0
    for row, n in enumerate(need):
        tables[row, :n] = order[at : at + n]
        at += n
    lengths.copy_(_int(lens + [0] * (rows - len(lens))))
    state.copy_(_int([0, blocks - at]))
    free[: blocks - at] = order[at:].sort().values
    references.zero_()
    return {"book": book, "before": book.clone(), "tables": tables, "lengths": lengths, "state": state, "free": free, "references": references,
            "status": torch.zeros(1, dtype=torch.int32, device=DEVICE),
            "pools": [_randn(gen, blocks, case["kv_heads"], case["block"], case["dim"]) for _ in range(2 * case["layers"])]}


def _fork_inputs(case, gen):
    lens, children = _lengths(case, "context", case["lo"], case["hi"]), case["children"]
    parents = len(lens)
    blocks = math.ceil(sum(-(-n // case["block"]) for n in lens) * 1.25) + parents * children + 1
    parent = [p for p in range(parents) for _ in range(children)]
    return {**_book(case, gen, lens, parents * (1 + children), blocks), "parent": _int(parent), "child": _int([parents + i for i in range(len(parent))]),
            "done": _int(list(range(parents)))}


def _compact_inputs(case, gen):
    lens = _lengths(case, "context", case["lo"], case["hi"])
    blocks = math.ceil(sum(-(-n // case["block"]) for n in lens) * (1 + case["spare"])) + 1
    return {**_book(case, gen, lens, len(lens), blocks), "max_moves": blocks // 2}


_INPUTS = {"cache": _cache_inputs, "decode": _decode_inputs, "prefill": _prefill_inputs, "fork": _fork_inputs, "compact": _compact_inputs}


# --------------------------------------------------------------------------- the framework's operators


def _ops():
    package = os.path.join(os.getcwd(), "qwen3.6-2080ti_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import hip_ops

    return hip_ops


def _own_cache(s):
    case, ops = s["case"], _ops()
    ops.paged_kv8_append(s["key"], s["value"], s["keys"], s["values"], s["slots"], case["block"])
    return ops.paged_kv8_gather(s["keys"], s["values"], s["tables"], case["prefix"] + case["new"], case["block"])


def _own_decode(s):
    return _ops().paged_attention_decode_kv8(s["query"], s["tables"], s["keys"], s["values"], s["lens"], s["case"]["block"], gate=s["gate"])


def _own_prefill(s):
    return _ops().paged_attention_prefill_kv8(s["query"], s["cu"], s["prefix"], s["keys"], s["values"], s["tables"], s["case"]["block"], max_new=s["max_new"], gate=s["gate"])


def _own_fork(s):
    ops = _ops()
    s["book"].copy_(s["before"])
    copies = ops.paged_kv_fork(s["tables"], s["lengths"], s["parent"], s["child"], s["free"], s["state"], s["references"], s["status"], s["case"]["block"])
    ops.paged_kv_copy(s["pools"], copies.sources, copies.targets)
    ops.paged_kv_release(s["tables"], s["lengths"], s["done"], s["free"], s["state"], s["references"], s["status"])
    return {"book": s["book"], "status": s["status"], "sources": copies.sources, "targets": copies.targets, "pools": s["pools"]}


def _own_compact(s):
    ops = _ops()
    s["book"].copy_(s["before"])
    copies = ops.paged_kv_compact(s["tables"], s["free"], s["state"], s["references"], s["status"], max_moves=s["max_moves"])
    ops.paged_kv_copy(s["pools"], copies.sources, copies.targets)
    return {"book": s["book"], "status": s["status"], "sources": copies.sources, "targets": copies.targets, "pools": s["pools"]}


_OWN = {"cache": _own_cache, "decode": _own_decode, "prefill": _own_prefill, "fork": _own_fork, "compact": _own_compact}


# --------------------------------------------------------------------------- plain forms


def _places(case, slots, is_key):
    """Places in the flat pool of the bytes of tokens in slots (tokens,): codes (tokens, kv_heads, D), scales (tokens, kv_heads)."""
    bs, dim, heads = case["block"], case["dim"], case["kv_heads"]
    t = (slots % 16)[:, None]
    tile = (slots // bs)[:, None] * heads + torch.arange(heads, device=slots.device)  # (tokens, heads)
    run = (tile * (bs // 16) + (slots % bs // 16)[:, None]) * 16 * (dim + 1)
    d = torch.arange(dim, device=slots.device)
    if is_key:
        code = ((d // 16) * 16 + t) * 16 + d % 16
    else:
        code = (((d // 64 * 4 + t // 4) * 16 + d // 4 % 16) * 4 + d % 4) * 4 + t % 4
    return run[..., None] + code[:, None], run + 16 * dim


def _read(case, pool, slots, is_key):
    """The codes' values and the scale bytes of the tokens in slots: (tokens, kv_heads, D) fp32 and (tokens, kv_heads)."""
    code_at, scale_at = _places(case, slots, is_key)
    flat = pool.view(torch.uint8).view(-1)
    return flat[code_at].view(torch.float8_e4m3fn).float(), flat[scale_at].int()


def _values(case, pool, slots, is_key):
    codes, byte = _read(case, pool, slots, is_key)
    return torch.ldexp(codes, byte[..., None] - 127)


def _write(case, pool, slots, x, is_key):
    x = x.float()
    runs, which = torch.unique(slots // 16, return_inverse=True)
    shape = (runs.numel(), case["kv_heads"])
    top = torch.zeros(shape, device=DEVICE).scatter_reduce_(0, which[:, None].expand(-1, shape[1]), x.abs().amax(-1), "amax")
    first = torch.full(shape[:1], 16, dtype=torch.int64, device=DEVICE).scatter_reduce_(0, which, slots % 16, "amin")
    every = (runs[:, None] * 16 + torch.arange(16, device=DEVICE)).view(-1)
    codes, old = _read(case, pool, every, is_key)
    old = old.view(-1, 16, case["kv_heads"])[:, 0]
    byte = torch.where(first[:, None] > 0, torch.maximum(old, _least(top)), _least(top))
    codes = torch.ldexp(codes.view(-1, 16, *codes.shape[1:]), torch.where(first[:, None] > 0, old - byte, 0)[:, None, :, None]).flatten(0, 1)
    flat = pool.view(torch.uint8).view(-1)
    code_at, scale_at = _places(case, every, is_key)
    flat[code_at] = codes.to(torch.float8_e4m3fn).view(torch.uint8)
    flat[scale_at.view(-1, 16, case["kv_heads"])[:, 0]] = byte.to(torch.uint8)
    flat[_places(case, slots, is_key)[0]] = torch.ldexp(x, 127 - byte[which][..., None]).to(torch.float8_e4m3fn).view(torch.uint8)


def _plain_cache(s):
    case = s["case"]
    bs, valid = case["block"], case["prefix"] + case["new"]
    at = torch.arange(valid, device=DEVICE)
    slots = (s["tables"].long()[:, at // bs] * bs + at % bs).reshape(-1)
    out = []
    for new, pool, is_key in ((s["key"], s["keys"], True), (s["value"], s["values"], False)):
        _write(case, pool, s["slots"], new, is_key)
        out.append(_values(case, pool, slots, is_key).view(case["batch"], valid, case["kv_heads"], case["dim"]).transpose(1, 2).bfloat16().contiguous())
    return out


def _row(s, row, length):
    """Keys and values (kv_heads, length, D) fp32 of a row."""
    bs = s["case"]["block"]
    at = torch.arange(length, device=DEVICE)
    slots = s["tables"][row].long()[at // bs] * bs + at % bs
    return [_values(s["case"], s[pool], slots, pool == "keys").transpose(0, 1).contiguous() for pool in ("keys", "values")]


def _plain_decode(s):
    case = s["case"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    out = torch.empty((case["batch"], heads, 1, dim), dtype=torch.float32, device=DEVICE)
    for row, length in enumerate(_lengths(case, "context", case["lo"], case["hi"])):
        keys, values = _row(s, row, length)
        q = s["query"][row].float().view(kv_heads, heads // kv_heads, dim)
        for g in range(kv_heads):
            scores = q[g] @ keys[g].T * dim**-0.5
            e = torch.exp(scores - scores.amax(-1, keepdim=True))
            out[row, g * q.shape[1] : (g + 1) * q.shape[1], 0] = (e / e.sum(-1, keepdim=True)) @ values[g]
    if s["gate"] is not None:
        out = out / (1 + torch.exp(-s["gate"].float()))[:, :, None]
    return out.bfloat16()


def _plain_prefill(s):
    case = s["case"]
    heads, dim = case["heads"], case["dim"]
    group = heads // case["kv_heads"]
    out = torch.empty(s["query"].shape, dtype=torch.float32, device=DEVICE)
    lo = 0
    for row, (n, p) in enumerate(zip(s["new"], s["lens"])):
        keys, values = _row(s, row, p + n)
        hidden = torch.arange(p + n, device=DEVICE)[None] > p + torch.arange(n, device=DEVICE)[:, None]
        for h in range(heads):
            scores = torch.where(hidden, -math.inf, s["query"][lo : lo + n, h].float() @ keys[h // group].T * dim**-0.5)
            e = torch.exp(scores - scores.amax(-1, keepdim=True))
            out[lo : lo + n, h] = (e / e.sum(-1, keepdim=True)) @ values[h // group]
        lo += n
    if s["gate"] is not None:
        out = out / (1 + torch.exp(-s["gate"].float()))
    return out.bfloat16()


def _copy_pages(s, sources, targets):
    there = sources >= 0
    source, target = sources[there].long(), targets[there].long()
    for pool in s["pools"]:
        pool[target] = pool[source]


def _set_free(s, is_free):
    ids = is_free.nonzero().view(-1).int()
    s["free"].fill_(-1)
    s["free"][: ids.numel()] = ids
    s["state"][0] = 0
    s["state"][1] = ids.numel()


def _is_free(s):
    head, count = s["state"].tolist()
    is_free = torch.zeros(s["free"].shape, dtype=torch.bool, device=DEVICE)
    is_free[s["free"][head : head + count].long()] = True
    return is_free


def _plain_fork(s):
    s["book"].copy_(s["before"])
    bs, tables, lengths = s["case"]["block"], s["tables"], s["lengths"]
    # fork
    parent, child = s["parent"].long(), s["child"].long()
    length = lengths[parent].long()
    full, partly = length // bs, length % bs > 0
    nth = partly.long().cumsum(0) - partly.long()
    fresh = s["free"][(s["state"][0] + nth).clamp(max=s["free"].numel() - 1)]
    rows = tables[parent]
    last = rows.gather(1, full[:, None])[:, 0]
    sources, targets = torch.where(partly, last, -1), torch.where(partly, fresh, -1)
    shared = rows[torch.arange(rows.shape[1], device=DEVICE) < full[:, None]].long()
    s["references"].add_(torch.bincount(shared, minlength=s["references"].numel()).int())
    rows.scatter_(1, full[:, None], targets[:, None])
    tables[child] = rows
    lengths[child] = length.int()
    taken = partly.sum().int()
    s["state"].add_(torch.stack((taken, -taken)))
    _copy_pages(s, sources, targets)
    # free
    done = s["done"].long()
    ids = tables[done].view(-1)
    left = s["references"] - torch.bincount(ids[ids >= 0].long(), minlength=s["references"].numel()).int()
    tables[done] = -1
    lengths[done] = 0
    s["references"].copy_(left.clamp(min=0))
    _set_free(s, _is_free(s) | (left < 0))
    s["status"].zero_()
    return {"book": s["book"], "status": s["status"], "sources": sources, "targets": targets, "pools": s["pools"]}


def _plain_compact(s):
    s["book"].copy_(s["before"])
    is_free = _is_free(s)
    blocks = is_free.numel()
    held = torch.zeros_like(is_free)
    held[s["tables"][s["tables"] >= 0].long()] = True
    source, target = held.nonzero().view(-1).flip(0), is_free.nonzero().view(-1)
    n = min(source.numel(), target.numel(), s["max_moves"])
    source, target = source[:n], target[:n]
    n = int((source > target).sum())  # they stay apart in order: the first n
    source, target = source[:n], target[:n]
    place = torch.arange(blocks, dtype=torch.int32, device=DEVICE)
    place[source] = target.int()
    s["tables"].copy_(torch.where(s["tables"] >= 0, place[s["tables"].clamp(min=0).long()], s["tables"]))
    s["references"][target] = s["references"][source]
    s["references"][source] = 0
    is_free[target] = False
    is_free[source] = True
    _set_free(s, is_free)
    sources = torch.full((s["max_moves"],), -1, dtype=torch.int32, device=DEVICE)
    targets = sources.clone()
    sources[:n] = source.int()
    targets[:n] = target.int()
    _copy_pages(s, sources, targets)
    s["status"].zero_()
    return {"book": s["book"], "status": s["status"], "sources": sources, "targets": targets, "pools": s["pools"]}


_PLAIN = {"cache": _plain_cache, "decode": _plain_decode, "prefill": _plain_prefill, "fork": _plain_fork, "compact": _plain_compact}


# --------------------------------------------------------------------------- what each has to read, write and compute


def _work_cache(case):
    tokens, each = case["batch"] * case["new"], case["kv_heads"] * case["dim"]
    dense = case["batch"] * (case["new"] + case["prefix"])
    # a key and a value, two bytes each on one side and one on the other
    return {"bytes": (tokens + dense) * each * 6, "flops": 0}


def _work_decode(case):
    total = sum(_lengths(case, "context", case["lo"], case["hi"]))
    row = case["heads"] * case["dim"]
    return {"bytes": total * case["kv_heads"] * case["dim"] * 2 + case["batch"] * row * (6 if case["gated"] else 4), "flops": 4 * row * total}


def _work_prefill(case):
    new, prefix = _new_and_prefix(case)
    row = case["heads"] * case["dim"]
    keys = sum(new) + sum(prefix)
    return {"bytes": keys * case["kv_heads"] * case["dim"] * 2 + sum(new) * row * (6 if case["gated"] else 4),
            "flops": sum(4 * row * (n * p + n * (n + 1) // 2) for n, p in zip(new, prefix))}


def _page(case):
    return 2 * case["layers"] * case["kv_heads"] * case["block"] * case["dim"] * 2


def _work_fork(case):
    lens, bs = _lengths(case, "context", case["lo"], case["hi"]), case["block"]
    entries = sum(-(-n // bs) for n in lens)
    copies = case["children"] * sum(n % bs > 0 for n in lens)
    blocks = math.ceil(entries * 1.25) + case["batch"] * case["children"] + 1
    # pages read and written; table entries read once and written for each child; references; the list read and written
    return {"bytes": 2 * copies * _page(case) + entries * (1 + case["children"]) * 4 + entries * 8 + 2 * blocks * 4, "flops": 0}


def _work_compact(case):
    need = sum(-(-n // case["block"]) for n in _lengths(case, "context", case["lo"], case["hi"]))
    blocks = math.ceil(need * (1 + case["spare"])) + 1
    moves = round(need * (1 - need / blocks))  # of blocks at random places, those past the last of a packed cache
    return {"bytes": 2 * moves * _page(case) + 2 * need * 4 + 2 * blocks * 4, "flops": 0}


_WORK = {"cache": _work_cache, "decode": _work_decode, "prefill": _work_prefill, "fork": _work_fork, "compact": _work_compact}


# --------------------------------------------------------------------------- the same in 64 bits


def _e4m3(byte):
    """The values in 64 bits of E4M3 bytes: sign, four bits of exponent with a bias of 7, three of mantissa."""
    byte = byte.long()
    exponent, mantissa = byte // 8 % 16, byte % 8
    size = torch.where(exponent == 0, mantissa.double() * 2.0**-9, (8 + mantissa).double() * torch.exp2(exponent.double() - 10))
    size = torch.where(byte % 128 == 127, math.nan, size)
    return torch.where(byte < 128, size, -size)


def _unpack(case, blocks, is_key):
    """The values (n, kv_heads, block_size, D) in 64 bits of pool blocks (n, kv_heads, bytes), and the exponents (n, kv_heads, runs)."""
    n, heads, dim, bs = blocks.shape[0], blocks.shape[1], case["dim"], case["block"]
    runs = blocks.view(n, heads, bs // 16, -1)
    codes = runs[..., : 16 * dim].contiguous()
    if is_key:
        codes = codes.view(n, heads, -1, dim // 64, 4, 16, 16).permute(0, 1, 2, 5, 3, 4, 6)
    else:
        codes = codes.view(n, heads, -1, dim // 64, 4, 16, 4, 4).permute(0, 1, 2, 4, 7, 3, 5, 6)
    exponent = runs[..., 16 * dim].double() - 127
    values = _e4m3(codes.reshape(n, heads, bs // 16, 16 * dim)) * torch.exp2(exponent)[..., None]
    return values.view(n, heads, bs, dim), exponent


def _exact_cache(s):
    case = s["case"]
    batch, new, prefix, heads, dim, bs = case["batch"], case["new"], case["prefix"], case["kv_heads"], case["dim"], case["block"]
    valid = new + prefix
    need = -(-valid // bs)
    start = prefix // 16 * 16  # the first run that is written
    out = []
    for pool, x, is_key in ((s["keys"], s["key"], True), (s["values"], s["value"], False)):
        result = torch.empty((batch, heads, valid, dim), dtype=torch.float64, device=DEVICE)
        for row in range(batch):
            dense, exponent = _unpack(case, pool.view(torch.uint8)[s["tables"][row, :need].long()], is_key)
            dense = dense.transpose(0, 1).reshape(heads, need * bs, dim)
            exponent = exponent.transpose(0, 1).reshape(heads, -1)
            dense[:, prefix:valid] = x[row * new : (row + 1) * new].double().transpose(0, 1)
            dense[:, valid:] = 0
            runs = dense[:, start:].reshape(heads, -1, 16, dim)
            fresh = (torch.arange(start, need * bs, device=DEVICE) >= prefix).view(-1, 16, 1)
            top = (runs * fresh).abs().amax((-1, -2))
            e = torch.ceil(torch.log2(top / 448)).clamp(-117, 120)
            if prefix % 16:
                e[:, 0] = torch.maximum(e[:, 0], exponent[:, start // 16])
            e = e[..., None, None]
            # a step of the grid is 2^-3 of the value's power of two, and 2^-9 of the scale at least
            step = torch.exp2(torch.maximum(torch.floor(torch.log2(runs.abs())) - 3, e - 9))
            dense[:, start:] = (torch.round(runs / step) * step).view(heads, -1, dim)
            result[row] = dense[:, :valid]
        out.append(result)
    return out


def _exact_kv(s, row, length):
    case = s["case"]
    ids = s["tables"][row, : -(-length // case["block"])].long()
    both = []
    for name in ("keys", "values"):
        pool = s[name].view(torch.uint8)
        dense = torch.cat([_unpack(case, pool.index_select(0, part), name == "keys")[0] for part in ids.split(1024)])
        both.append(dense.transpose(0, 1).reshape(case["kv_heads"], -1, case["dim"])[:, :length].contiguous())
    return both


def _exact_decode(s):
    case = s["case"]
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device=DEVICE)
    for row, length in enumerate(s["lens"].tolist()):
        keys, values = _exact_kv(s, row, length)
        for h in range(case["heads"]):
            g = h // (case["heads"] // case["kv_heads"])
            p = torch.softmax(keys[g] @ s["query"][row, h, 0].double() / math.sqrt(case["dim"]), dim=0)
            out[row, h, 0] = p @ values[g]
    return out if s["gate"] is None else out * torch.sigmoid(s["gate"].double())[:, :, None]


def _exact_prefill(s):
    case = s["case"]
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device=DEVICE)
    cu, prefix = s["cu"].tolist(), s["prefix"].tolist()
    group = case["heads"] // case["kv_heads"]
    for row, p in enumerate(prefix):
        keys, values = _exact_kv(s, row, p + cu[row + 1] - cu[row])
        for lo in range(cu[row], cu[row + 1], 512):
            hi = min(cu[row + 1], lo + 512)
            seen = p + hi - cu[row]
            last = p - cu[row] + torch.arange(lo, hi, device=DEVICE)
            hidden = torch.arange(seen, device=DEVICE)[None] > last[:, None]
            for h in range(case["heads"]):
                scores = (s["query"][lo:hi, h].double() @ keys[h // group, :seen].T / math.sqrt(case["dim"])).masked_fill(hidden, -math.inf)
                out[lo:hi, h] = torch.softmax(scores, dim=-1) @ values[h // group, :seen]
    return out if s["gate"] is None else out * torch.sigmoid(s["gate"].double())


def _exact_books(s, tables, lengths, free, references, sources, targets):
    """What a pass over pages returns, from lists; the pools' pages copied one by one."""
    blocks = s["free"].numel()
    book = [i for row in tables for i in row] + lengths + [0, len(free)] + free + [-1] * (blocks - len(free)) + references
    for pool in s["pools"]:
        for source, target in zip(sources, targets):
            if source >= 0:
                pool[target] = pool[source]
    return {"book": _int(book), "status": _int([0]), "sources": _int(sources), "targets": _int(targets), "pools": [pool.double() for pool in s["pools"]]}


def _exact_fork(s):
    bs = s["case"]["block"]
    tables, lengths, references = s["tables"].tolist(), s["lengths"].tolist(), s["references"].tolist()
    free = s["free"].tolist()[: s["state"].tolist()[1]]
    sources, targets = [], []
    for parent, child in zip(s["parent"].tolist(), s["child"].tolist()):
        lengths[child] = lengths[parent]
        sources.append(-1)
        targets.append(-1)
        for i in range(-(-lengths[parent] // bs)):
            tables[child][i] = tables[parent][i]
            if (i + 1) * bs <= lengths[parent]:
                references[tables[parent][i]] += 1
            else:
                sources[-1] = tables[parent][i]
                targets[-1] = tables[child][i] = free.pop(0)
    for row in s["done"].tolist():
        for i, block in enumerate(tables[row]):
            if block < 0:
                continue
            if references[block] > 0:
                references[block] -= 1
            else:
                free.append(block)
            tables[row][i] = -1
        lengths[row] = 0
    return _exact_books(s, tables, lengths, sorted(free), references, sources, targets)


def _exact_compact(s):
    tables, lengths, references = s["tables"].tolist(), s["lengths"].tolist(), s["references"].tolist()
    free = s["free"].tolist()[: s["state"].tolist()[1]]
    sources, targets = [], []
    for source in sorted({i for row in tables for i in row if i >= 0}, reverse=True):
        if len(sources) == min(s["max_moves"], len(free)) or free[len(sources)] > source:
            break
        sources.append(source)
        targets.append(free[len(targets)])
    place = dict(zip(sources, targets))
    tables = [[place.get(i, i) for i in row] for row in tables]
    for source, target in place.items():
        references[source], references[target] = 0, references[source]
    free = sorted(free[len(targets) :] + sources)
    pad = [-1] * (s["max_moves"] - len(sources))
    return _exact_books(s, tables, lengths, free, references, sources + pad, targets + pad)


_EXACT = {"cache": _exact_cache, "decode": _exact_decode, "prefill": _exact_prefill, "fork": _exact_fork, "compact": _exact_compact}
