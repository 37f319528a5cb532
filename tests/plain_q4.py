"""The 4-bit cache format stated plainly for tests, in numpy, without code of ``axon_b200``: steps
from a table of all step values, rows placed in pages by loops."""

from __future__ import annotations

import numpy as np

GROUP, TOP, NAN_BYTE = 16, 223, 255


def step_of(byte: int) -> float:
    """The step a byte stands for: five exponent and three mantissa bits, subnormal below 8."""
    if byte == NAN_BYTE:
        return float("nan")
    e, m = int(byte) >> 3, int(byte) & 7
    return m * 2.0 ** -17 if e == 0 else (8 + m) * 2.0 ** (e - 18)


STEPS = np.array([step_of(b) for b in range(TOP + 1)])


def quantise(x: np.ndarray):
    """Float32 rows [..., w] to (nibbles [..., w] in 0..15, step bytes [..., w / 16])."""
    g = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, GROUP)
    top = np.abs(g).max(-1)                                    # (NaN wins in numpy's max)
    fine = np.isfinite(top)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        t = top * np.float32(2.0 / 15.0)                       # one rounding to 32 bits
        byte = np.minimum(np.searchsorted(STEPS, np.where(fine, t, 0.0).astype(np.float64), side="left"), TOP)
        s = STEPS[byte].astype(np.float32)
        inv = np.where(s > 0, np.float32(1) / s, np.float32(0))
        c = np.clip(np.rint(g * inv[..., None]), -7, 7)
    c = np.where(fine[..., None], c, 0).astype(np.int64) + 8
    return c.reshape(x.shape).astype(np.uint8), np.where(fine, byte, NAN_BYTE).astype(np.uint8)


def values(nibbles: np.ndarray, steps: np.ndarray) -> np.ndarray:
    """What nibbles and step bytes stand for, in float64."""
    s = np.array([step_of(b) for b in range(256)])[steps.astype(np.int64)]
    c = nibbles.astype(np.float64).reshape(*nibbles.shape[:-1], -1, GROUP) - 8
    return (c * s[..., None]).reshape(nibbles.shape)


def parts(page_size: int, head_dim: int, v_dim: int, planes: int):
    """(offset, row bytes) of key codes, key steps, value codes, value steps in a head's record, and its bytes."""
    at, out = 0, []
    for width in (head_dim, v_dim)[:planes]:
        for row in (width // 2, width // 16):
            out.append((at, row))
            at += -(-page_size * row // 16) * 16
    return out, at


def put(pool: np.ndarray, page: int, entry: int, kv_head: int, record: int, place, in_page: int, row: np.ndarray) -> None:
    """Writes ``row`` bytes of one position into ``pool [pages][entries][bytes]``."""
    at = kv_head * record + place[0] + in_page * place[1]
    pool[page, entry, at:at + place[1]] = row


def codes_of(nibbles: np.ndarray) -> np.ndarray:
    return nibbles[..., 0::2] | (nibbles[..., 1::2] << 4)


def store_row(pool, table, slot, pos, entry, kv_head, page_size, head_dim, v_dim, planes, k, v) -> None:
    """Quantises one position's key and value row of a kv head into the pool, through the block table."""
    places, record = parts(page_size, head_dim, v_dim, planes)
    page, i = int(table[slot, pos // page_size]), pos % page_size
    for x, p in ((k, places[:2]), (v, places[2:])):
        if x is None or not p:
            continue
        n, s = quantise(x)
        put(pool, page, entry, kv_head, record, p[0], i, codes_of(n))
        put(pool, page, entry, kv_head, record, p[1], i, s)


def attention(q, k, v, positions, window, scale):
    """softmax(q k scale) v for one kv head in float64: q [rows, hd] at ``positions``, k and v [T, width]; and
    the parts that an error bound needs (weights times |v|, and the largest sum of |q k| of each row)."""
    s = (q @ k.T) * scale
    t = np.arange(k.shape[0])
    hidden = t[None] > positions[:, None]
    if window:
        hidden |= t[None] <= positions[:, None] - window
    s[hidden] = -np.inf
    w = np.exp(s - s.max(-1, keepdims=True))
    w /= w.sum(-1, keepdims=True)
    size = np.where(hidden, 0, (np.abs(q) @ np.abs(k).T) * abs(scale)).max(-1)
    seen = np.where(hidden.all(0)[:, None], 0, v)
    return w @ seen, w @ np.abs(seen), size
