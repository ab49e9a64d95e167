"""A full-attention layer over a KV cache held in 4 bits, operator by operator, as cases that can be timed and checked.

* ``plan``      block tables and slot maps of a step, built on the GPU from the requests' lengths
* ``prologue``  q/k RMSNorm, rotary embedding of several position axes, and the K/V write through the slot map
* ``cache``     K/V quantised into the 4-bit cache through the slot map, and the cache's dense view
* ``decode``    one token per sequence over the 4-bit cache
* ``prefill``   a prompt, or a chunk of one, over the 4-bit cache, with the output gate

The 4-bit cache.  A group is 32 consecutive dims of one token and KV head.  It is held as a scale 2^e, one byte e + 127,
and 32 E2M1 codes (sign, and 0 0.5 1 1.5 2 3 4 6).  e is the least integer with max |x| <= 7 2^e, within [-125, 125];
x / 2^e goes to the nearest value, ties to the even code, and saturates at 6.  A group that is not finite has the byte
255 and reads as NaN.  The pools are uint8 ``(blocks, kv_heads, block_size * 17 * D / 32)``: per block and head, runs of
16 tokens, each first the codes (16 D / 2 bytes, even dim in the low half of its byte), then the scales (16 D / 32):

* keys    codes  [group D/32][token 16][16 bytes];        scales [group % 4][token 16][group / 4]
* values  codes  [pair of token % 4][token / 4][dim / (D/16)][token within the pair][D/32 bytes], a "pair" being
          512 / D tokens;                                  scales [group][token 16]

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
EPS = 1e-6
THETA = 10_000_000.0


def listed() -> list[dict]:
    return [
        # The plan of one decode step of a full batch: 128 conversations take one token each.
        _plan("plan_step", batch=128, new_lo=1, new_hi=1, prefix_lo=256, prefix_hi=32768),
        # Admission of many ragged prompts at once, the token arrays padded to what the server allows in a step.
        _plan("plan_prompts", batch=61, new_lo=1, new_hi=8192, prefix_lo=0, prefix_hi=700, pad=1000),
        # The norm, rotary and write launch of a full decode batch, text far into its context.
        _prologue("prologue_step", tokens=128, image=0, start=100_000),
        # The same for a prefill chunk of pages with pictures, heads of 128 rotated whole.
        _prologue("prologue_images", tokens=5003, image=23, start=0, heads=16, kv_heads=4, dim=128, sections=(16, 24, 24), interleaved=False),
        # One token for each of five short conversations, and the cache read back dense, as a caller without paging does.
        _cache("cache_step", batch=5, new=1, prefix=333),
        # A prompt written in one go and read back.
        _cache("cache_prompt", batch=3, new=4001, prefix=0),
        # The smallest call of a chat server: four short conversations.
        _decode("decode_few", batch=4, lo=512, hi=512),
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
    ]


def draw(rng: random.Random) -> dict:
    family = rng.choice(("plan", "prologue", "cache", "decode", "decode", "prefill", "prefill"))
    block = rng.choice((16, 16, 32, 64))
    index = rng.choice(("int32", "int64"))
    if family == "plan":
        batch = _log_int(rng, 1, 300)
        new_hi = _log_int(rng, 1, max(1, 200_000 // batch))
        return _plan(None, batch=batch, new_lo=rng.randint(0, new_hi), new_hi=new_hi, prefix_lo=0, prefix_hi=_log_int(rng, 1, 32768),
                     block=block, pad=rng.choice((0, 0, 37, 2000)))
    if family == "prologue":
        heads, kv_heads, dim, sections, interleaved = rng.choice((
            (16, 2, 256, (11, 11, 10), True), (16, 2, 256, (11, 11, 10), True), (16, 4, 128, (16, 24, 24), False), (8, 2, 128, (16, 8, 8), True), (4, 4, 256, (32,), False)))
        return _prologue(None, tokens=_log_int(rng, 1, 5000), image=rng.choice((0, 5, 23)), start=_log_int(rng, 1, 200_000), heads=heads, kv_heads=kv_heads,
                         dim=dim, sections=sections, interleaved=interleaved, block=block, index=index)
    if family == "cache":
        heads_dim = rng.choice(((2, 256), (2, 128), (4, 128), (1, 256)))
        new = _log_int(rng, 1, 4000)
        return _cache(None, batch=rng.randint(1, 3), new=new, prefix=rng.choice((0, _log_int(rng, 1, 4001 - new))), kv_heads=heads_dim[0], dim=heads_dim[1], block=block, index=index)
    if family == "decode":
        heads, kv_heads, dim = rng.choice(((16, 2, 256), (16, 2, 256), (8, 2, 128), (16, 1, 128), (6, 2, 256), (12, 2, 128), (16, 1, 256)))
        hi = _log_int(rng, 1, 32768)
        return _decode(None, batch=_log_int(rng, 1, 64), lo=_log_int(rng, 1, hi), hi=hi, heads=heads, kv_heads=kv_heads, dim=dim, block=block, gated=rng.random() < 0.5,
                       index=index)
    heads, kv_heads, dim = rng.choice(((16, 2, 256), (16, 2, 256), (8, 2, 128), (4, 4, 256), (20, 4, 128), (16, 1, 128)))
    tokens = _log_int(rng, 24, 4096)
    batch = rng.randint(1, max(1, min(8, tokens // 24)))
    new_hi = max(1, tokens // batch)
    prefix_hi = rng.choice((0, _log_int(rng, 16, 8192)))
    return _prefill(None, batch=batch, new_lo=rng.randint(max(1, new_hi // 4), new_hi), new_hi=new_hi, prefix_lo=prefix_hi // 3, prefix_hi=prefix_hi, heads=heads,
                    kv_heads=kv_heads, dim=dim, block=block, gated=rng.random() < 0.7, index=index)


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _case(name, family, values) -> dict:
    case = {"family": family, **values}
    if name is not None:
        case["name"] = name
    return case


def _plan(name, *, batch, new_lo, new_hi, prefix_lo, prefix_hi, block=16, pad=0):
    return _case(name, "plan", dict(batch=batch, new_lo=new_lo, new_hi=new_hi, prefix_lo=prefix_lo, prefix_hi=prefix_hi, block=block, pad=pad))


def _prologue(name, *, tokens, image, start, heads=16, kv_heads=2, dim=256, sections=(11, 11, 10), interleaved=True, block=16, index="int32"):
    return _case(name, "prologue", dict(tokens=tokens, image=image, start=start, heads=heads, kv_heads=kv_heads, dim=dim, sections=",".join(map(str, sections)),
                                        interleaved=interleaved, block=block, index=index))


def _cache(name, *, batch, new, prefix, kv_heads=2, dim=256, block=16, index="int32"):
    return _case(name, "cache", dict(batch=batch, new=new, prefix=prefix, kv_heads=kv_heads, dim=dim, block=block, index=index))


def _decode(name, *, batch, lo, hi, heads=16, kv_heads=2, dim=256, block=16, gated=True, index="int32"):
    return _case(name, "decode", dict(batch=batch, lo=lo, hi=hi, heads=heads, kv_heads=kv_heads, dim=dim, block=block, gated=gated, index=index))


def _prefill(name, *, batch, new_lo, new_hi, prefix_lo, prefix_hi, heads=16, kv_heads=2, dim=256, block=16, gated=True, index="int32"):
    return _case(name, "prefill", dict(batch=batch, new_lo=new_lo, new_hi=new_hi, prefix_lo=prefix_lo, prefix_hi=prefix_hi, heads=heads, kv_heads=kv_heads, dim=dim,
                                       block=block, gated=gated, index=index))


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


def _pack(x, is_key):
    """A 4-bit pool (blocks, kv_heads, bytes) that holds x (blocks, kv_heads, block_size, dim)."""
    n, h, bs, d = x.shape
    g = x.float().view(n, h, bs // 16, 16, d // 32, 32)
    mant, expo = torch.frexp(g.abs().amax(-1))  # amax = mant 2^expo, mant in [0.5, 1)
    e = (expo - 3 + (mant > 0.875)).clamp(-125, 125)  # 7 2^(expo-3) = 0.875 2^expo
    a = torch.ldexp(g, -e[..., None])
    code = torch.bucketize(a.abs(), torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=x.device))  # ties to the lower code ...
    for tie, up in ((0.75, 2), (1.75, 4), (3.5, 6)):  # ... which is the odd one here
        code = torch.where(a.abs() == tie, up, code)
    code = (code + 8 * (a < 0)).to(torch.uint8)
    codes = code[..., 0::2] | (code[..., 1::2] << 4)  # (n, h, run, token, group, 16 bytes)
    scales = (e + 127).to(torch.uint8)  # (n, h, run, token, group)
    if is_key:
        codes = codes.permute(0, 1, 2, 4, 3, 5)
        scales = scales.view(n, h, bs // 16, 16, d // 128, 4).permute(0, 1, 2, 5, 3, 4)
    else:
        tpc = 512 // d
        codes = codes.reshape(n, h, bs // 16, 4, 4 // tpc, tpc, 16, d // 32).permute(0, 1, 2, 4, 3, 6, 5, 7)
        scales = scales.transpose(3, 4)
    flat = torch.cat((codes.reshape(n, h, bs // 16, -1), scales.reshape(n, h, bs // 16, -1)), dim=-1)
    return flat.reshape(n, h, -1)


def _pools(case, gen, blocks):
    pools = []
    for is_key in (True, False):
        pool = torch.empty((blocks, case["kv_heads"], case["block"] * 17 * case["dim"] // 32), dtype=torch.uint8, device=DEVICE)
        scale = _channels(gen, case["kv_heads"], case["dim"]) if is_key else 1.0
        for lo in range(0, blocks, 8192):
            n = min(blocks - lo, 8192)
            pool[lo : lo + n] = _pack(_randn(gen, n, case["kv_heads"], case["block"], case["dim"], dtype=torch.float32) * scale, is_key)
        pools.append(pool)
    return pools


def _plan_inputs(case, gen):
    new, prefix = _new_and_prefix(case)
    bs, batch = case["block"], case["batch"]
    want = [(n + p + bs - 1) // bs for n, p in zip(new, prefix)]
    have = [(p + bs - 1) // bs for p in prefix]
    blocks = math.ceil(sum(want) * 1.25) + 8
    order = torch.randperm(blocks, generator=gen, device=DEVICE).to(torch.int32)
    tables = torch.full((batch, max(want) + 3), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for row, n in enumerate(have):
        tables[row, :n] = order[at : at + n]
        at += n
    free = torch.full((blocks,), -1, dtype=torch.int32, device=DEVICE)
    free[: blocks - at] = order[at:].sort().values
    # lengths and the free list's cursor side by side, so that a pass sets both back with one copy
    step = _int(prefix + [0, blocks - at])
    return {"tables": tables, "step": step, "before": step.clone(), "lengths": step[:batch], "free_state": step[batch:], "free": free, "counts": _int(new),
            "status": torch.zeros(1, dtype=torch.int32, device=DEVICE), "max_tokens": sum(new) + case["pad"]}


def _prologue_inputs(case, gen):
    tokens, heads, kv_heads, dim = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    sections = [int(x) for x in case["sections"].split(",")]
    rng = random.Random(f"{tokens} {case['image']}")
    axes, at = [], case["start"]
    while len(axes) < tokens:  # words, then a picture: one time, a grid of rows and columns
        for _ in range(rng.randint(3, 60)):
            axes.append((at,) * 3)
            at += 1
        if case["image"]:
            high, wide = rng.randint(2, case["image"]), rng.randint(2, case["image"])
            axes += [(at, at + r, at + c) for r in range(high) for c in range(wide)]
            at += max(high, wide)
    positions = _int(list(zip(*axes[:tokens]))[: len(sections)], _index(case))
    blocks = -(-tokens // case["block"]) + 7
    order = torch.randperm(blocks, generator=gen, device=DEVICE)
    token = torch.arange(tokens, device=DEVICE)
    slots = order[token // case["block"]] * case["block"] + token % case["block"]
    shape = (blocks, kv_heads, case["block"], dim)
    return {"q_proj": _randn(gen, tokens, heads, 2 * dim), "k_proj": _randn(gen, tokens, kv_heads, dim), "v_proj": _randn(gen, tokens, kv_heads, dim),
            "q_norm": 0.2 * _randn(gen, dim), "k_norm": 0.2 * _randn(gen, dim), "positions": positions, "slots": slots, "sections": sections,
            "keys": _randn(gen, *shape), "values": _randn(gen, *shape)}


def _cache_inputs(case, gen):
    new, prefix, kv_heads, dim, bs = case["new"], case["prefix"], case["kv_heads"], case["dim"], case["block"]
    tables, blocks = _tables(gen, [new + prefix] * case["batch"], bs, _index(case))
    keys, values = _pools(case, gen, blocks)
    at = prefix + torch.arange(new, device=DEVICE)
    slots = (tables.long()[:, at // bs] * bs + at % bs).reshape(-1)
    tokens = slots.numel()
    return {"key": (_randn(gen, tokens, kv_heads, dim, dtype=torch.float32) * _channels(gen, kv_heads, dim).view(kv_heads, dim)).bfloat16(),
            "value": _randn(gen, tokens, kv_heads, dim), "keys": keys, "values": values, "tables": tables, "slots": slots}


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


_INPUTS = {"plan": _plan_inputs, "prologue": _prologue_inputs, "cache": _cache_inputs, "decode": _decode_inputs, "prefill": _prefill_inputs}


# --------------------------------------------------------------------------- the framework's operators


def _ops():
    package = os.path.join(os.getcwd(), "qwen3.6-2080ti_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import hip_ops

    return hip_ops


def _own_plan(s):
    s["step"].copy_(s["before"])
    plan = _ops().paged_kv_plan(s["tables"], s["lengths"], s["counts"], s["free"], s["free_state"], s["status"], s["case"]["block"], max_tokens=s["max_tokens"])
    return {"tables": s["tables"], "step": s["step"], "status": s["status"], "cu": plan.cu_seqlens, "starts": plan.starts, "positions": plan.positions, "slots": plan.slots}


def _own_prologue(s):
    query, _ = _ops().qk_norm_mrope_kv_append(
        s["q_proj"], s["k_proj"], s["v_proj"], s["q_norm"], s["k_norm"], s["positions"], s["sections"], s["keys"], s["values"], s["slots"], s["case"]["block"], eps=EPS,
        rope_theta=THETA, interleaved=s["case"]["interleaved"])
    return query, s["keys"], s["values"]


def _own_cache(s):
    case, ops = s["case"], _ops()
    ops.paged_kv4_append(s["key"], s["value"], s["keys"], s["values"], s["slots"], case["block"])
    return ops.paged_kv4_gather(s["keys"], s["values"], s["tables"], case["prefix"] + case["new"], case["block"])


def _own_decode(s):
    return _ops().paged_attention_decode_kv4(s["query"], s["tables"], s["keys"], s["values"], s["lens"], s["case"]["block"], gate=s["gate"])


def _own_prefill(s):
    return _ops().paged_attention_prefill_kv4(s["query"], s["cu"], s["prefix"], s["keys"], s["values"], s["tables"], s["case"]["block"], max_new=s["max_new"], gate=s["gate"])


_OWN = {"plan": _own_plan, "prologue": _own_prologue, "cache": _own_cache, "decode": _own_decode, "prefill": _own_prefill}


# --------------------------------------------------------------------------- plain forms


def _plain_plan(s):
    s["step"].copy_(s["before"])
    bs, tables, width = s["case"]["block"], s["tables"], s["tables"].shape[1]
    lengths, counts = s["lengths"].long(), s["counts"].long()
    have, want = (lengths + bs - 1) // bs, (lengths + counts + bs - 1) // bs
    need = want - have
    first = s["free_state"][0] + need.cumsum(0) - need
    column = torch.arange(width, device=DEVICE)
    fresh = (column >= have[:, None]) & (column < want[:, None])
    ids = s["free"][(first[:, None] + column - have[:, None]).clamp(0, s["free"].numel() - 1)]
    tables.copy_(torch.where(fresh, ids, tables))
    end = counts.cumsum(0)
    begin = end - counts
    token = torch.arange(s["max_tokens"], device=DEVICE)
    row = torch.searchsorted(end, token, right=True).clamp(max=counts.numel() - 1)
    live = token < end[-1]
    position = torch.where(live, lengths[row] + token - begin[row], -1)
    slot = torch.where(live, tables[row, (position // bs).clamp(min=0)].long() * bs + position % bs, -1)
    starts = lengths.int()
    s["status"].copy_((need.sum() > s["free_state"][1]).int())
    s["lengths"].add_(s["counts"])
    s["free_state"].add_(torch.stack((need.sum(), -need.sum())).int())
    cu = torch.cat((torch.zeros(1, dtype=torch.int64, device=DEVICE), end)).int()
    return {"tables": tables, "step": s["step"], "status": s["status"], "cu": cu, "starts": starts, "positions": position.int(), "slots": slot}


def _axis(sections, interleaved):
    """The position axis of each frequency: the sections one after the other, or turn by turn (axis a at j = a, a + n, a + 2n ..
    for as many as its section has, the first axis elsewhere)."""
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    axis = [0] * sum(sections)
    for a in range(1, len(sections)):
        for j in range(a, min(len(sections) * sections[a], len(axis)), len(sections)):
            axis[j] = a
    return axis


def _norm_rotate(x, weight, cos, sin):
    y = x.float()
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * (1.0 + weight.float())
    half = cos.shape[-1]
    a, b = y[..., :half], y[..., half : 2 * half]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, y[..., 2 * half :]), dim=-1).bfloat16()


def _plain_prologue(s):
    case = s["case"]
    half = sum(s["sections"])
    freq = THETA ** (-torch.arange(half, device=DEVICE, dtype=torch.float64) / half)
    angle = s["positions"].double()[torch.tensor(_axis(s["sections"], case["interleaved"]), device=DEVICE)].T * freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    query = _norm_rotate(s["q_proj"][..., : case["dim"]], s["q_norm"], cos, sin)
    block, at = s["slots"] // case["block"], s["slots"] % case["block"]
    s["keys"][block, :, at] = _norm_rotate(s["k_proj"], s["k_norm"], cos, sin)
    s["values"][block, :, at] = s["v_proj"]
    return query, s["keys"], s["values"]


def _byte_places(case, slots, is_key):
    """Places in the flat pool of the bytes of tokens in slots (tokens,): codes (tokens, kv_heads, D/2), scales (tokens, kv_heads, D/32)."""
    bs, dim, heads = case["block"], case["dim"], case["kv_heads"]
    t = slots % 16
    base = (slots // bs)[:, None] * heads + torch.arange(heads, device=slots.device)  # (tokens, heads)
    base = (base * (bs // 16) + (slots % bs // 16)[:, None]) * (17 * dim // 2)
    byte = torch.arange(dim // 2, device=slots.device)
    group = torch.arange(dim // 32, device=slots.device)
    t = t[:, None]
    if is_key:
        code, scale = (byte // 16 * 16 + t) * 16 + byte % 16, (group % 4 * 16 + t) * (dim // 128) + group // 4
    else:
        each, pair = dim // 32, 512 // dim
        code = (((t % 4 // pair * 4 + t // 4) * 16 + byte // each) * pair + t % 4 % pair) * each + byte % each
        scale = group * 16 + t
    return base[..., None] + code[:, None], base[..., None] + (8 * dim + scale)[:, None]


_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _read(case, pool, slots, is_key):
    """The values (tokens, kv_heads, D) fp32 of the tokens in slots."""
    code_at, scale_at = _byte_places(case, slots, is_key)
    flat = pool.view(-1)
    codes = flat[code_at].int()
    table = torch.tensor(_VALUES + tuple(-v for v in _VALUES), device=DEVICE)
    both = torch.stack((table[codes & 15], table[codes >> 4]), dim=-1).view(*codes.shape[:2], -1, 32)
    return (both * torch.exp2(flat[scale_at].float() - 127)[..., None]).flatten(2)


def _write(case, pool, slots, x, is_key):
    x = x.float().view(*x.shape[:2], -1, 32)
    top = x.abs().amax(-1)
    e = (torch.floor(torch.log2(top.double())) - 2).clamp(-300, 300)
    e = (e + (top.double() > 7 * torch.exp2(e))).clamp(-125, 125)
    a = (x.double() * torch.exp2(-e)[..., None]).abs()
    code = (a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5) + 8 * (x < 0)
    code = code.to(torch.uint8)
    code_at, scale_at = _byte_places(case, slots, is_key)
    pool.view(-1)[code_at] = (code[..., 0::2] | (code[..., 1::2] << 4)).flatten(2)
    pool.view(-1)[scale_at] = (e + 127).to(torch.uint8)


def _plain_cache(s):
    case = s["case"]
    bs, valid = case["block"], case["prefix"] + case["new"]
    at = torch.arange(valid, device=DEVICE)
    slots = (s["tables"].long()[:, at // bs] * bs + at % bs).reshape(-1)
    out = []
    for new, pool, is_key in ((s["key"], s["keys"], True), (s["value"], s["values"], False)):
        _write(case, pool, s["slots"], new, is_key)
        out.append(_read(case, pool, slots, is_key).view(case["batch"], valid, case["kv_heads"], case["dim"]).transpose(1, 2).bfloat16().contiguous())
    return out


def _row(s, row, length):
    """Keys and values (kv_heads, length, D) fp32 of a row."""
    bs = s["case"]["block"]
    at = torch.arange(length, device=DEVICE)
    slots = s["tables"][row].long()[at // bs] * bs + at % bs
    return [_read(s["case"], s[pool], slots, pool == "keys").transpose(0, 1).contiguous() for pool in ("keys", "values")]


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


_PLAIN = {"plan": _plain_plan, "prologue": _plain_prologue, "cache": _plain_cache, "decode": _plain_decode, "prefill": _plain_prefill}


# --------------------------------------------------------------------------- what each has to read, write and compute


def _work_plan(case):
    new, prefix = _new_and_prefix(case)
    bs = case["block"]
    fresh = sum((n + p + bs - 1) // bs - (p + bs - 1) // bs for n, p in zip(new, prefix))
    # lengths read and written, counts, cu, starts; ids read and written; positions and slots
    return {"bytes": case["batch"] * 5 * 4 + fresh * 8 + (sum(new) + case["pad"]) * 12, "flops": 0}


def _work_prologue(case):
    return {"bytes": 2 * case["tokens"] * case["dim"] * (case["heads"] + 2 * case["kv_heads"]) * 2, "flops": 0}


def _work_cache(case):
    tokens, each = case["batch"] * case["new"], case["kv_heads"] * case["dim"]
    dense = case["batch"] * (case["new"] + case["prefix"])
    return {"bytes": (tokens + dense) * each * 81 // 16, "flops": 0}


def _work_decode(case):
    total = sum(_lengths(case, "context", case["lo"], case["hi"]))
    row = case["heads"] * case["dim"]
    return {"bytes": total * case["kv_heads"] * case["dim"] * 17 // 16 + case["batch"] * row * (6 if case["gated"] else 4), "flops": 4 * row * total}


def _work_prefill(case):
    new, prefix = _new_and_prefix(case)
    row = case["heads"] * case["dim"]
    keys = sum(new) + sum(prefix)
    return {"bytes": keys * case["kv_heads"] * case["dim"] * 17 // 16 + sum(new) * row * (6 if case["gated"] else 4),
            "flops": sum(4 * row * (n * p + n * (n + 1) // 2) for n, p in zip(new, prefix))}


_WORK = {"plan": _work_plan, "prologue": _work_prologue, "cache": _work_cache, "decode": _work_decode, "prefill": _work_prefill}


# --------------------------------------------------------------------------- the same in 64 bits


def _exact_plan(s):
    case = s["case"]
    bs, tables, free = case["block"], s["tables"].tolist(), iter(s["free"].tolist())
    lengths, counts = s["lengths"].tolist(), s["counts"].tolist()
    cu, positions, slots, taken = [0], [], [], 0
    for row, (length, n) in enumerate(zip(lengths, counts)):
        for position in range(length, length + n):
            if position % bs == 0:
                tables[row][position // bs] = next(free)
                taken += 1
            positions.append(position)
            slots.append(tables[row][position // bs] * bs + position % bs)
        cu.append(len(slots))
    pad = [-1] * (s["max_tokens"] - len(slots))
    head, count = s["free_state"].tolist()
    step = [length + n for length, n in zip(lengths, counts)] + [head + taken, count - taken]
    return {"tables": _int(tables), "step": _int(step), "status": _int([0]), "cu": _int(cu), "starts": _int(lengths), "positions": _int(positions + pad),
            "slots": _int(slots + pad, torch.int64)}


def _exact_prologue(s):
    case = s["case"]
    sections, half = s["sections"], sum(s["sections"])
    positions = s["positions"].double()

    def turned(x, weight):
        x = x.double()
        y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * (weight.double() + 1)
        for j in range(half):
            if case["interleaved"]:
                a = j % len(sections)
                a = a if j < len(sections) * sections[a] else 0
            else:
                a = next(i for i in range(len(sections)) if j < sum(sections[: i + 1]))
            turn = torch.polar(torch.ones_like(positions[a]), positions[a] * THETA ** (-j / half))
            z = torch.complex(y[..., j].clone(), y[..., j + half].clone()) * turn[:, None]
            y[..., j], y[..., j + half] = z.real, z.imag
        return y

    keys, values = s["keys"].double(), s["values"].double()
    for pool, new in ((keys, turned(s["k_proj"], s["k_norm"])), (values, s["v_proj"].double())):
        flat = pool.transpose(1, 2).reshape(-1, case["kv_heads"], case["dim"])
        flat[s["slots"]] = new
        pool.copy_(flat.view(pool.shape[0], case["block"], case["kv_heads"], case["dim"]).transpose(1, 2))
    return turned(s["q_proj"][..., : case["dim"]], s["q_norm"]), keys, values


def _unpack(case, blocks, is_key):
    """The values (n, kv_heads, block_size, D) in 64 bits of pool blocks (n, kv_heads, bytes)."""
    n, heads, dim = blocks.shape[0], blocks.shape[1], case["dim"]
    runs = blocks.view(n, heads, case["block"] // 16, 17 * dim // 2)
    codes, scales = runs[..., : 8 * dim], runs[..., 8 * dim :]
    if is_key:
        codes = codes.reshape(n, heads, -1, dim // 32, 16, 16).transpose(3, 4)
        scales = scales.reshape(n, heads, -1, 4, 16, dim // 128).permute(0, 1, 2, 4, 5, 3)
    else:
        pair = 512 // dim
        codes = codes.reshape(n, heads, -1, 4 // pair, 4, 16, pair, dim // 32).permute(0, 1, 2, 4, 3, 6, 5, 7)
        scales = scales.reshape(n, heads, -1, dim // 32, 16).transpose(3, 4)
    codes = codes.reshape(n, heads, case["block"], dim // 2).long()
    nibbles = torch.stack((codes % 16, codes // 16), dim=-1).flatten(3)
    size = nibbles % 8
    # E2M1: two exponent bits, one mantissa bit, the lowest exponent without the hidden one
    value = torch.where(size < 2, size * 0.5, (2 + size % 2).double() * torch.exp2((size // 2).double() - 2))
    value = torch.where(nibbles < 8, value, -value).view(n, heads, case["block"], -1, 32)
    exponent = scales.reshape(n, heads, case["block"], dim // 32, 1).double() - 127
    return (value * torch.exp2(exponent)).flatten(3)


def _nearest(x):
    """x (tokens, kv_heads, D) as the 4-bit cache holds it, in 64 bits."""
    x = x.double().view(*x.shape[:2], -1, 32)
    e = torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True) / 7)).clamp(-125, 125)
    grid = torch.tensor(_VALUES, dtype=torch.float64, device=DEVICE)
    distance = ((x * torch.exp2(-e)).abs()[..., None] - grid).abs()
    odd = torch.tensor([0, 1] * 4, device=DEVICE)
    best = torch.where(distance == distance.amin(-1, keepdim=True), odd, 2).argmin(-1)  # the even code of a tie
    return (torch.sign(x) * grid[best] * torch.exp2(e)).flatten(2)


def _exact_cache(s):
    case = s["case"]
    batch, new, prefix, heads, dim, bs = case["batch"], case["new"], case["prefix"], case["kv_heads"], case["dim"], case["block"]
    need = -(-(new + prefix) // bs)
    out = []
    for pool, x, is_key in ((s["keys"], s["key"], True), (s["values"], s["value"], False)):
        dense = _unpack(case, pool[s["tables"][:, :need].long().reshape(-1)], is_key)
        dense = dense.view(batch, need, heads, bs, dim).transpose(1, 2).reshape(batch, heads, need * bs, dim)[:, :, : new + prefix].contiguous()
        at = 0
        for row in range(batch):
            for lo in range(0, new, 512):
                n = min(512, new - lo)
                dense[row, :, prefix + lo : prefix + lo + n] = _nearest(x[at : at + n]).transpose(0, 1)
                at += n
        out.append(dense)
    return out


def _exact_kv(s, row, length):
    case = s["case"]
    ids = s["tables"][row, : -(-length // case["block"])].long()
    both = []
    for name in ("keys", "values"):
        dense = torch.cat([_unpack(case, s[name].index_select(0, part), name == "keys") for part in ids.split(1024)])
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


_EXACT = {"plan": _exact_plan, "prologue": _exact_prologue, "cache": _exact_cache, "decode": _exact_decode, "prefill": _exact_prefill}
