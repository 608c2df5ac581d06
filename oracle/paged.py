"""The paged operators in numpy, 64 bits, token by token: rotary positions, a cache of microscaled codes in pages and
attention over it. Arrays as ``ancha_amd.paged`` has them: codes [2, pages, heads, page, bytes], scales
[2, pages, heads, page, dim / 32]; a batch is (starts, lengths, table), and a page number outside the cache is a page
that is not there.
"""
from __future__ import annotations

import numpy as np

from . import mx


def rotate(x: np.ndarray, positions, freqs, layout: str = "half", magnitude: float = 1.0) -> np.ndarray:
    """x [rows, heads, dim] at its rows' positions, by complex numbers."""
    x = x.astype(np.float64).copy()
    n = len(freqs)
    first = slice(0, n) if layout == "half" else slice(0, 2 * n, 2)
    second = slice(n, 2 * n) if layout == "half" else slice(1, 2 * n, 2)
    turn = magnitude * np.exp(1j * np.asarray(positions, np.float64)[:, None, None] * np.asarray(freqs, np.float64))
    z = (x[..., first] + 1j * x[..., second]) * turn
    x[..., first], x[..., second] = z.real, z.imag
    return x


def rows_of(batch, rows: int):
    """(row, sequence, position) of each row that is of a sequence."""
    starts, lengths, _ = batch
    for i, length in enumerate(lengths):
        for r in range(starts[i], min(starts[i + 1], rows)):
            yield r, i, int(length) - int(starts[i + 1]) + r


def place(batch, i: int, position: int, pages: int, page: int):
    """(page, slot) of a token, or None."""
    table = batch[2]
    if position < 0 or position // page >= table.shape[1]:
        return None
    at = int(table[i, position // page])
    return (at, position % page) if 0 <= at < pages else None


def write(codes, scales, fmt: str, k, v, batch) -> None:
    """Rows k, v [rows, heads, dim] (keys already turned) into their places."""
    _, pages, heads, page, size = codes.shape
    dim = k.shape[2]
    both = [mx.encode(x.reshape(-1, dim), fmt) for x in (k, v)]
    for r, i, position in rows_of(batch, k.shape[0]):
        to = place(batch, i, position, pages, page)
        if to is None:
            continue
        for which, (c, s) in enumerate(both):
            codes[which, to[0], :, to[1]] = c[r * heads:(r + 1) * heads, :size]
            scales[which, to[0], :, to[1]] = s[r * heads:(r + 1) * heads, :dim // 32]


def sequence(codes, scales, fmt: str, batch, i: int, size: int):
    """(keys, values) [size, heads, dim] of sequence i, and which tokens are there; zeros where they are not."""
    _, pages, heads, page, _ = codes.shape
    dim = 32 * scales.shape[4]
    out, there = np.zeros((2, size, heads, dim)), np.zeros(size, bool)
    for t in range(min(size, int(batch[1][i]))):
        at = place(batch, i, t, pages, page)
        if at is None:
            continue
        there[t] = True
        for which in (0, 1):
            c = np.zeros((heads, mx.padded(dim) // (1 if fmt == "fp8" else 2)), np.uint8)
            s = np.zeros((heads, mx.padded(dim) // 32), np.uint8)
            c[:, :codes.shape[4]], s[:, :dim // 32] = codes[which, at[0], :, at[1]], scales[which, at[0], :, at[1]]
            out[which, t] = mx.decode(c, s, fmt, dim)
    return out[0], out[1], there


def attention(q, codes, scales, fmt: str, batch, scale=None, causal: bool = True, window=None):
    """([rows, heads, dim] result, sums over keys of weight |v| and of |v|, largest scale sum |q k|) of q in 64 bits."""
    q = q.astype(np.float64)
    rows, heads, dim = q.shape
    kv = codes.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    out, size, total, reach = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape), np.zeros((rows, heads, 1))
    held = {}
    for r, i, position in rows_of(batch, rows):
        if i not in held:
            held[i] = sequence(codes, scales, fmt, batch, i, max(0, int(batch[1][i])))
        k, v, there = held[i]
        at = np.arange(k.shape[0])
        sees = there & (at <= position if causal else True) & (at > position - window if window else True)
        if not sees.any():
            continue
        for h in range(heads):
            key, value = k[sees, h * kv // heads], v[sees, h * kv // heads]
            with np.errstate(invalid="ignore"):
                s = scale * (key @ q[r, h])
                w = np.exp(s - s.max())
                w /= w.sum()
                out[r, h] = w @ value
                size[r, h], total[r, h] = w @ np.abs(value), np.abs(value).sum(0)
                reach[r, h] = scale * (np.abs(key) @ np.abs(q[r, h])).max()
    return out, size, total, reach
