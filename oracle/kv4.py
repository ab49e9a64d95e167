"""The 4-bit KV cache and what stands on it, restated on the CPU in 64 bits: number format, tile layout, step plan,
rotary embedding of several position axes, and attention.  The reference has no counterpart; the checks are the
format's landmarks, the layout formulas byte by byte, and textbook softmax attention."""

from __future__ import annotations

import math
from typing import Sequence

import numpy as np

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def scale_exponent(amax: float) -> int:
    """The least e in [-125, 125] with amax <= 7 2^e (the largest where there is none)."""
    e = -125
    while e < 125 and amax > 7.0 * 2.0**e:
        e += 1
    return e


def quantize_group(x: np.ndarray) -> tuple[int, list[int]]:
    """Scale byte and the 32 codes of a group."""
    x = np.asarray(x, dtype=np.float64)
    if not np.all(np.isfinite(x)):
        return 255, [0] * len(x)
    e = scale_exponent(float(np.max(np.abs(x))))
    codes = []
    for v in x:
        a = abs(float(v)) * 2.0**-e
        gaps = [abs(a - g) for g in GRID]
        best = min(range(8), key=lambda i: (gaps[i], i % 2))
        codes.append(best + (8 if v < 0 else 0))
    return e + 127, codes


def dequantize_group(byte: int, codes: Sequence[int]) -> np.ndarray:
    if byte == 255:
        return np.full(len(codes), np.nan)
    return np.array([(-1.0 if c & 8 else 1.0) * GRID[c & 7] * 2.0 ** (byte - 127) for c in codes])


def quantized(x: np.ndarray) -> np.ndarray:
    """x (.., D) as the cache holds it; vectorised :func:`quantize_group` and back."""
    x = np.asarray(x, dtype=np.float64)
    g = x.reshape(-1, 32)
    out = np.full_like(g, np.nan)
    ok = np.isfinite(g).all(1)
    amax = np.abs(g[ok]).max(1)
    e = np.full(amax.shape, -125.0)
    with np.errstate(divide="ignore"):
        e = np.clip(np.ceil(np.log2(amax / 7.0)), -125, 125)
    a = np.abs(g[ok]) * 2.0 ** -e[:, None]
    gaps = np.abs(a[..., None] - np.array(GRID))
    best = np.lexsort((np.broadcast_to(np.array([0, 1] * 4), gaps.shape), gaps), axis=-1)[..., 0]  # nearest, then even
    out[ok] = np.sign(g[ok]) * np.array(GRID)[best] * 2.0 ** e[:, None]
    return out.reshape(x.shape)


def tile_bytes(dim: int, block: int) -> int:
    return block * 17 * dim // 32


def key_place(dim: int, token: int, group: int) -> tuple[int, int]:
    """Byte offsets in a tile of a token's 16 key code bytes of a group, and of its scale."""
    run, t = divmod(token, 16)
    base = run * 17 * dim // 2
    return base + (group * 16 + t) * 16, base + 8 * dim + ((group % 4) * 16 + t) * (dim // 128) + group // 4


def value_places(dim: int, token: int, group: int) -> tuple[list[int], int]:
    """Byte offsets of the group's 16 value code bytes, and of its scale."""
    run, t = divmod(token, 16)
    base = run * 17 * dim // 2
    pair, each = 512 // dim, dim // 32
    q, r = divmod(t, 4)
    places = []
    for d in range(32 * group, 32 * group + 32, 2):
        chunk, inside = divmod(d, dim // 16)
        places.append(base + (((r // pair * 4 + q) * 16 + chunk) * pair + r % pair) * each + inside // 2)
    return places, base + 8 * dim + group * 16 + t


def write(pool: np.ndarray, slot: int, head: int, block: int, x: np.ndarray, is_key: bool) -> None:
    """One head's values x (D,) into slot of a uint8 pool (P, H_kv, tile)."""
    dim = len(x)
    if slot < 0 or slot >= pool.shape[0] * block:
        return
    tile = pool[slot // block, head]
    for g in range(dim // 32):
        byte, codes = quantize_group(x[32 * g : 32 * g + 32])
        pairs = [codes[i] | codes[i + 1] << 4 for i in range(0, 32, 2)]
        if is_key:
            at, scale = key_place(dim, slot % block, g)
            places = range(at, at + 16)
        else:
            places, scale = value_places(dim, slot % block, g)
        for place, b in zip(places, pairs):
            tile[place] = b
        tile[scale] = byte


def read(pool: np.ndarray, slot: int, head: int, block: int, dim: int, is_key: bool) -> np.ndarray:
    tile = pool[slot // block, head]
    out = np.empty(dim)
    for g in range(dim // 32):
        if is_key:
            at, scale = key_place(dim, slot % block, g)
            places = range(at, at + 16)
        else:
            places, scale = value_places(dim, slot % block, g)
        codes = [c for place in places for c in (int(tile[place]) & 15, int(tile[place]) >> 4)]
        out[32 * g : 32 * g + 32] = dequantize_group(int(tile[scale]), codes)
    return out


def plan(tables: list[list[int]], lengths: list[int], counts: list[int], free: list[int], head: int, count: int, block: int, max_tokens: int, capacity: int):
    """(status, tables, lengths, head, count, cu, starts, positions, slots) of a step, row by row and token by token."""
    empty = [-1] * max_tokens
    refused = lambda code: (code, tables, lengths, head, count, [0] * (len(lengths) + 1), list(lengths), empty, empty)  # noqa: E731
    if head < 0 or count < 0 or head + count > capacity:
        return refused(3)
    if any(n < 0 or length < 0 or length + n > 2**31 - 1 - block for length, n in zip(lengths, counts)):
        return refused(4)
    want = [-(-(length + n) // block) for length, n in zip(lengths, counts)]
    need = [w - -(-length // block) for w, length in zip(want, lengths)]
    if any(w > len(row) for w, row in zip(want, tables)):
        return refused(2)
    if sum(need) > count:
        return refused(1)
    if sum(counts) > max_tokens:
        return refused(5)
    tables = [list(row) for row in tables]
    ids = iter(free[head : head + sum(need)])
    cu, positions, slots = [0], [], []
    for row, (length, n) in enumerate(zip(lengths, counts)):
        for lb in range(-(-length // block), want[row]):
            tables[row][lb] = next(ids)
        for p in range(length, length + n):
            positions.append(p)
            block_id = tables[row][p // block]
            slots.append(-1 if block_id < 0 else block_id * block + p % block)
        cu.append(len(positions))
    pad = [-1] * (max_tokens - len(positions))
    return 0, tables, [length + n for length, n in zip(lengths, counts)], head + sum(need), count - sum(need), cu, list(lengths), positions + pad, slots + pad


def mrope_axis(j: int, sections: Sequence[int], interleaved: bool) -> int:
    n = len(sections)
    if interleaved:
        a = j % n
        return a if j < n * sections[a] else 0
    for a in range(n):
        if j < sum(sections[: a + 1]):
            return a
    raise ValueError(j)


def norm_mrope(x: np.ndarray, weight: np.ndarray, positions: np.ndarray, sections: Sequence[int], interleaved: bool, theta: float, eps: float) -> np.ndarray:
    """x (tokens, heads, D): RMSNorm with (1 + w), then each pair (j, j + half) turned by its axis's position."""
    x = np.asarray(x, dtype=np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (1.0 + np.asarray(weight, dtype=np.float64))
    half = sum(sections)
    for j in range(half):
        angle = positions[mrope_axis(j, sections, interleaved)].astype(np.float64) * theta ** (-j / half)
        # the product is rounded to 2^-53 of its size: fine up to positions of 2^30
        turned = (y[..., j] + 1j * y[..., j + half]) * np.exp(1j * angle)[:, None]
        y[..., j], y[..., j + half] = turned.real, turned.imag
    return y


def _round_to(x: np.ndarray, bits: int, least: float) -> np.ndarray:
    """x to the nearest number of ``bits`` significant bits and no place below ``least``, ties to even."""
    place = np.maximum(2.0 ** (np.floor(np.log2(np.maximum(np.abs(x), 1e-300))) - (bits - 1)), least)
    return np.rint(x / place) * place


def query_pieces(row: np.ndarray) -> tuple[np.ndarray, np.ndarray, float]:
    """A bf16 query row (D,) as the scores take it: hi, lo and a power of two ``scale``, the row being about ``scale (hi +
    lo / 16)``.  The largest element lies in [128, 256) over the scale; hi is E4M3 (4 bits, places down to 2^-9) of the
    element on a grid of 2^-10 of the power of two at the largest of its eight dims as E4M3 rounds it; lo is E4M3 of 16
    times what is left."""
    row = np.asarray(row, dtype=np.float64)
    top = np.abs(row).max()
    if top == 0.0:
        return row, row, 1.0
    scale = 2.0 ** (math.floor(math.log2(top)) - 7)
    y = row / scale
    eight = np.repeat(np.abs(y).reshape(-1, 8).max(1), 8)
    grid = 2.0 ** (np.floor(np.log2(np.maximum(_round_to(eight, 4, 2.0**-140), 1e-300))) - 10)
    hi = _round_to(np.rint(y / grid) * grid, 4, 2.0**-9)
    return hi, _round_to((y - hi) * 16, 4, 2.0**-9), scale


def attention(q: np.ndarray, keys: np.ndarray, values: np.ndarray, seen: np.ndarray, scale: float) -> np.ndarray:
    """One query head (D,) over keys/values (T, D) where seen (T,) holds; zeros where it sees nothing."""
    if not seen.any():
        return np.zeros_like(q, dtype=np.float64)
    s = keys[seen] @ q * scale
    p = np.exp(s - s.max())
    return (p / p.sum()) @ values[seen]


def sigmoid(x: np.ndarray) -> np.ndarray:
    return 1.0 / (1.0 + np.exp(-np.asarray(x, dtype=np.float64)))


def default_scale(dim: int) -> float:
    return 1.0 / math.sqrt(dim)
