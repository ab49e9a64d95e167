"""The 8-bit KV cache restated on the CPU in 64 bits: number format, tile layout, and what a call writes.  The reference has no
counterpart; the checks are the format's landmarks and the layout formulas byte by byte."""

from __future__ import annotations

import numpy as np

RUN = 16


def value(byte: int) -> float:
    """The value of an E4M3 byte: sign, four bits of exponent with a bias of 7, three of mantissa; 0x7f and 0xff are NaN."""
    exponent, mantissa = byte >> 3 & 15, byte & 7
    if byte & 127 == 127:
        return float("nan")
    size = mantissa * 2.0**-9 if exponent == 0 else (8 + mantissa) * 2.0 ** (exponent - 10)
    return -size if byte & 128 else size


GRID = np.array([value(b) for b in range(127)])
VALUES = np.array([value(b) for b in range(256)])


def scale_exponent(amax: float) -> int:
    """The least e in [-117, 120] with amax <= 448 2^e (the largest where there is none)."""
    e = -117
    while e < 120 and amax > 448.0 * 2.0**e:
        e += 1
    return e


def encode(x: np.ndarray, e: int) -> np.ndarray:
    """The nearest code of x / 2^e, ties to the even one, but 240 for 256 at the largest scale; a NaN where x is not finite."""
    x = np.asarray(x, dtype=np.float64)
    ok = np.isfinite(x)
    a = np.where(ok, np.abs(x), 0.0) * 2.0**-e
    up = np.clip(np.searchsorted(GRID, a), 1, 126)  # GRID[up - 1] <= a <= GRID[up] within the range
    below, above = a - GRID[up - 1], GRID[up] - a
    code = np.where((below < above) | ((below == above) & (up % 2 == 1)), up - 1, up)
    if e == 120:
        code = np.minimum(code, 0x77)
    return np.where(ok, code + 128 * (np.signbit(x) & (code > 0)), 127).astype(np.uint8)


def tile_bytes(dim: int, block: int) -> int:
    return block // RUN * (RUN * dim + 16)


def code_places(dim: int, token: int, is_key: bool) -> np.ndarray:
    """Byte offsets in a run of a token's D codes."""
    d = np.arange(dim)
    if is_key:
        return d // 64 * 1024 + d // 16 % 4 * 256 + token * 16 + d % 16
    return d // 64 * 1024 + token // 4 * 256 + d // 4 % 16 * 16 + d % 4 * 4 + token % 4


def _run(pool: np.ndarray, slot: int, head: int, block: int, dim: int) -> np.ndarray:
    """The bytes of the run that a slot lies in."""
    at = slot % block // RUN * (RUN * dim + 16)
    return pool[slot // block, head, at : at + RUN * dim + 16]


def append(pool: np.ndarray, slots: np.ndarray, rows: np.ndarray, block: int, is_key: bool) -> None:
    """One call: rows (tokens, heads, D) into the slots of pool (blocks, heads, tile bytes), in place."""
    tokens, heads, dim = rows.shape
    runs: dict[int, list[int]] = {}
    for n, slot in enumerate(int(s) for s in slots):
        if 0 <= slot < pool.shape[0] * block:
            runs.setdefault(slot // RUN, []).append(n)
    for run, members in runs.items():
        for head in range(heads):
            at = _run(pool, run * RUN, head, block, dim)
            new = {int(slots[n]) % RUN: rows[n, head] for n in members}
            every = np.concatenate(list(new.values()))
            finite = np.abs(every[np.isfinite(every)])
            byte = scale_exponent(float(finite.max()) if finite.size else 0.0) + 127
            first = min(new)
            if first > 0:
                old = min(max(int(at[RUN * dim]), 10), 247)
                byte = max(byte, old)
                if byte > old:
                    for t in range(first):
                        places = code_places(dim, t, is_key)
                        at[places] = encode(VALUES[at[places]] * 2.0 ** (old - byte), 0)
            for t, x in new.items():
                at[code_places(dim, t, is_key)] = encode(x, byte - 127)
            at[RUN * dim :] = 0
            at[RUN * dim] = byte


def read(pool: np.ndarray, slot: int, head: int, block: int, dim: int, is_key: bool) -> np.ndarray:
    """The values of the token in a slot."""
    at = _run(pool, slot, head, block, dim)
    return VALUES[at[code_places(dim, slot % RUN, is_key)]] * 2.0 ** (int(at[RUN * dim]) - 127)


def same_bytes(a: np.ndarray, b: np.ndarray, dim: int) -> bool:
    """Whether two pools hold the same codes and scales; the sign of a zero or a NaN is free."""

    def plain(pool: np.ndarray) -> np.ndarray:
        runs = pool.reshape(-1, RUN * dim + 16).copy()
        codes = runs[:, : RUN * dim]
        codes[codes == 0x80] = 0
        codes[codes == 0xFF] = 0x7F
        return runs

    return np.array_equal(plain(a), plain(b))
