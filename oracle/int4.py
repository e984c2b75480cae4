"""4-bit KV pools in 64 bits: the format's definition, its layout byte by byte, and attention over what a pool holds."""

from __future__ import annotations

import numpy as np

BLOCK = 16          # slots of a block
MOST = 57344.0      # where elements saturate


def scale_of(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """Scale and zero point of rows [..., D] (float64, finite)."""
    lo, hi = np.minimum(x.min(-1), 0.0), np.maximum(x.max(-1), 0.0)
    step = (hi - lo) / 15.0
    _, exponent = np.frexp(step)                              # step = m * 2^exponent, m in [0.5, 1)
    unit = np.ldexp(1.0, np.maximum(exponent - 7, -20))       # of a number of 7 significant bits
    s = np.ceil(step / unit) * unit
    return s, np.where(s > 0, np.rint(-lo / np.where(s > 0, s, 1.0)), 0.0)


def quantise(x: np.ndarray) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """(codes, scales, zero points) of rows [..., D]; a code c stands for scale * (c - zero point)."""
    x = np.nan_to_num(x.astype(np.float64), nan=0.0, posinf=MOST, neginf=-MOST).clip(-MOST, MOST)
    s, z = scale_of(x)
    c = np.rint(x / np.where(s > 0, s, 1.0)[..., None]) + z[..., None]
    return c.clip(0, 15).astype(np.uint8), s, z


def block_bytes(hkv: int, d: int) -> int:
    return 2 * hkv * (8 * d + 32)


def places(hkv: int, d: int) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """Inside a block: byte and upper-half flag of the code of [slot, head, element], byte of the word of [slot, head]."""
    at = np.zeros((BLOCK, 2 * hkv, d), dtype=np.int64)
    upper = np.zeros((BLOCK, 2 * hkv, d), dtype=bool)
    word = np.zeros((BLOCK, 2 * hkv), dtype=np.int64)
    for t in range(BLOCK):
        for head in range(2 * hkv):
            word[t, head] = 16 * hkv * d + 2 * (head * BLOCK + t)
            for e in range(d):
                if head < hkv:
                    nibble = (e % 8) // 2 + (4 if e % 2 else 0)
                    byte = head * 8 * d + t * (d // 2) + (e // 8) * 4 + nibble // 2
                else:
                    columns, units = d // 16, d // 64
                    column, within = divmod(e, columns)
                    nibble, unit = divmod(within, units)
                    pair, half = divmod(t % 4, 2)
                    byte = head * 8 * d + (t // 4) * 2 * d + column * (d // 8) + (pair * units + unit) * 4 + half * 2 + nibble // 2
                at[t, head, e], upper[t, head, e] = byte, nibble % 2 == 1
    return at, upper, word


def decode_pool(pool: np.ndarray, hkv: int, d: int) -> tuple[np.ndarray, np.ndarray]:
    """float64 values [slots, 2 * Hkv, D] of a pool uint8 [slots, 2 * Hkv, D / 2 + 2], and the rows' scales."""
    at, upper, word = places(hkv, d)
    blocks = pool.reshape(-1, block_bytes(hkv, d))
    raw = blocks[:, at]
    code = np.where(upper, raw >> 4, raw & 15).astype(np.float64)
    bits = blocks[:, word].astype(np.uint16) | (blocks[:, word + 1].astype(np.uint16) << 8)
    s = (bits & 0xFFF0).view(np.float16).astype(np.float64)
    z = (bits & 15).astype(np.float64)
    with np.errstate(invalid="ignore"):
        values = (code - z[..., None]) * s[..., None]
    return values.reshape(-1, 2 * hkv, d), s.reshape(-1, 2 * hkv)


def store(pool: np.ndarray, slots, k: np.ndarray, v: np.ndarray) -> None:
    """Appends rows k, v [T, Hkv, D] to the pool, byte by byte; a slot outside it is skipped."""
    hkv, d = k.shape[1], k.shape[2]
    at, upper, word = places(hkv, d)
    code, s, z = quantise(np.concatenate([k, v], 1))
    bits = s.astype(np.float16).view(np.uint16) | z.astype(np.uint16)
    blocks = pool.reshape(-1, block_bytes(hkv, d))
    for i, slot in enumerate(slots):
        if not 0 <= slot < pool.shape[0]:
            continue
        block, t = blocks[slot // BLOCK], slot % BLOCK
        for mask, shift, pick in ((0xF0, 0, ~upper[t]), (0x0F, 4, upper[t])):
            block[at[t][pick]] = (block[at[t][pick]] & mask) | (code[i][pick] << shift)
        block[word[t]], block[word[t] + 1] = bits[i] & 255, bits[i] >> 8


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float, seen: np.ndarray):
    """Rows q [M, Hq, D] over keys k, v [N, Hkv, D], row m seeing the first seen[m] of them: (out, sum of p |v|), float64."""
    group = q.shape[1] // k.shape[1]
    out, size = np.zeros(q.shape), np.zeros(q.shape)
    hidden = np.arange(k.shape[0])[None, :] >= np.asarray(seen)[:, None]
    for h in range(q.shape[1]):
        x = (q[:, h].astype(np.float64) @ k[:, h // group].T) * scale
        x = np.where(hidden, -np.inf, x)
        top = x.max(-1, keepdims=True, initial=-np.inf)
        p = np.exp(x - np.where(np.isfinite(top), top, 0.0))
        total = p.sum(-1, keepdims=True)
        p = p / np.where(total > 0, total, 1.0)
        out[:, h], size[:, h] = p @ v[:, h // group], p @ np.abs(v[:, h // group])
    return out, size


def tokens_of(table_row, n: int, page_size: int) -> np.ndarray:
    """Slots of a sequence's first n tokens."""
    t = np.arange(n)
    return np.asarray(table_row)[t // page_size].astype(np.int64) * page_size + t % page_size
