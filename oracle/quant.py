"""float64 numpy restatement of the 8-bit K/V cache and the windowed read. Test infrastructure only.

e4m3: sign, exponent 2^-6 .. 2^8 with 3 mantissa bits, subnormals in steps of 2^-9, largest 448, 0x7f / 0xff NaN. A value
is code * 2^(x - 127), x the scale byte of its block.
"""
from __future__ import annotations

import math

import numpy as np

MIN_EXP = 17                       # scale bytes are at least 127 - 110
LARGEST = 1.875 * 2.0 ** 127


def decode_table() -> np.ndarray:
    """The 256 values of the codes."""
    out = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        out[c] = np.nan if c & 127 == 127 else -x if c & 128 else x
    return out


TABLE = decode_table()


def encode(y: np.ndarray) -> np.ndarray:
    """|y| <= 448 (or NaN) -> the nearest code's byte, ties to the even one; the sign of zero is kept."""
    grid = TABLE[:127]
    a = np.abs(y)
    hi = np.clip(np.searchsorted(grid, a), 1, 126)
    lo = hi - 1
    up = (a - grid[lo] > grid[hi] - a) | ((a - grid[lo] == grid[hi] - a) & (hi % 2 == 0))
    c = np.where(up, hi, lo)
    c = np.where(np.isnan(y), 127, c).astype(np.uint8)
    return c | np.where(np.signbit(y), 128, 0).astype(np.uint8)


def scale_byte(top: float) -> int:
    """The smallest x >= 17 with top <= 448 * 2^(x - 127)."""
    x = MIN_EXP
    if top > 0:
        x = max(x, math.ceil(math.log2(top / 448.0)) + 126)
    while x > MIN_EXP and top <= 448.0 * 2.0 ** (x - 128):
        x -= 1
    while top > 448.0 * 2.0 ** (x - 127):
        x += 1
    return x


def append(codes: np.ndarray, exps: np.ndarray, x: np.ndarray, starts, block: int) -> None:
    """Write x [B,G,T,d] at each sequence's start, in place (codes uint8 [B,G,C,d], exps uint8 [B,G,nb])."""
    B, G, C, _ = codes.shape
    T = x.shape[2]
    for b, start in enumerate(np.broadcast_to(starts, (B,))):
        start = int(start)
        for j in range(exps.shape[2]):
            lo, hi = j * block, min((j + 1) * block, C)
            n0, n1 = max(lo, start), min(hi, start + T)
            if n0 >= n1:
                continue
            for g in range(G):
                new = np.clip(x[b, g, n0 - start:n1 - start].astype(np.float64), -LARGEST, LARGEST)
                new = np.where(np.isfinite(x[b, g, n0 - start:n1 - start]), new, np.nan)
                fin = np.abs(new[np.isfinite(new)])
                e = scale_byte(float(fin.max()) if fin.size else 0.0)
                if start > lo:
                    was = int(exps[b, g, j])
                    e = max(e, was)
                    if e != was:
                        codes[b, g, lo:start] = encode(TABLE[codes[b, g, lo:start]] * 2.0 ** (was - e))
                codes[b, g, n0:n1] = encode(new * 2.0 ** (127 - e))
                exps[b, g, j] = e


def values(codes: np.ndarray, exps: np.ndarray, block: int) -> np.ndarray:
    s = 2.0 ** (exps.astype(np.float64) - 127)
    return TABLE[codes] * np.repeat(s, block, axis=2)[:, :, :codes.shape[2], None]


def visible(p: int, legal: int, window, sinks: int) -> np.ndarray:
    """The positions a query at p reads, ascending."""
    j = np.arange(min(legal, p + 1))
    return j if window is None else j[(j > p - window) | (j < sinks)]


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float) -> np.ndarray:
    """Softmax attention of one query q [h,d] over the rows k, v [n,d]; zeros for n == 0 and where no score is above
    -inf."""
    if k.shape[0] == 0:
        return np.zeros_like(q)
    with np.errstate(invalid="ignore"):
        s = (q @ k.T) * scale
        top = s.max(axis=-1, keepdims=True)
        w = np.exp(s - np.where(np.isneginf(top), 0.0, top))
        total = w.sum(axis=-1, keepdims=True)
        w = np.where(total == 0, 0.0, w / np.where(total == 0, 1.0, total))
        return w @ v


def range_attention(q: np.ndarray, k: np.ndarray, v: np.ndarray, legal, p0, window, sinks: int, scale: float):
    """q [B,G,h,T,d] at p0 + t (per sequence), over k, v [B,G,C,d] -> [B,G,h,T,d]."""
    B, G, h, T, d = q.shape
    out = np.zeros(q.shape)
    legal, p0 = np.broadcast_to(legal, (B,)), np.broadcast_to(p0, (B,))
    for b in range(B):
        for t in range(T):
            see = visible(int(p0[b]) + t, int(legal[b]), window, sinks)
            for g in range(G):
                out[b, g, :, t] = attend(q[b, g, :, t], k[b, g, see], v[b, g, see], scale)
    return out


def listed_attention(q: np.ndarray, k: np.ndarray, v: np.ndarray, rows: np.ndarray, scale: float) -> np.ndarray:
    """q [B,G,h,d] over the listed positions rows [B,G,S] (those outside [0, C) skipped) -> [B,G,h,d]."""
    B, G, h, d = q.shape
    out = np.zeros(q.shape)
    for b in range(B):
        for g in range(G):
            r = rows[b, g]
            r = r[(r >= 0) & (r < k.shape[2])]
            out[b, g] = attend(q[b, g], k[b, g, r], v[b, g, r], scale)
    return out
