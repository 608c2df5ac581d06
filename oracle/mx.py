"""Microscaled (MX) rows in numpy, 64 bits: blocks of 32 values along a row that share a power of two,
codes by the list of the format's values (nearest, ties to the even code, saturated).

For a block with largest magnitude a > 0 the scale byte is max(0, floor(log2 a) + 127 - E) with E = 8 for
e4m3 ("fp8") and 2 for e2m1 ("fp4"); a block of zeros has 0, one with a NaN or an infinity 255 and codes
0. Rows are stored as whole groups of 128 values, zeros behind the last one.
"""
from __future__ import annotations

import math

import numpy as np

BLOCK, GROUP = 32, 128
TOP = {"fp8": 8, "fp4": 2}


def grid(fmt: str) -> np.ndarray:
    """The non-negative values of the format in the order of their codes."""
    if fmt == "fp4":
        return np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
    values = [m * 2.0 ** -9 for m in range(8)]
    values += [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)]
    return np.array(values[:-1])  # the last code of each sign is the NaN


def padded(dim: int) -> int:
    return -(-dim // GROUP) * GROUP


def nearest(v: np.ndarray, fmt: str) -> np.ndarray:
    """Codes without sign of |v|."""
    g = grid(fmt)
    border = (g[1:] + g[:-1]) / 2
    size = np.abs(v)
    below, above = np.searchsorted(border, size, "left"), np.searchsorted(border, size, "right")
    return np.where(below % 2 == 0, below, above)


def scale_bytes(top: np.ndarray, fmt: str) -> np.ndarray:
    """Scale bytes of blocks whose largest magnitudes are `top` (not finite: 255)."""
    finite = np.isfinite(top)
    _, e = np.frexp(np.where(finite, top, 1.0))
    s = np.where(top > 0, np.maximum(e - 1 + 127 - TOP[fmt], 0), 0)
    return np.where(finite, s, 255).astype(np.uint8)


def encode(x: np.ndarray, fmt: str):
    """(codes, scales) as stored: x [rows, dim] of any float type."""
    rows, dim = x.shape
    full = np.zeros((rows, padded(dim)))
    full[:, :dim] = x
    blocks = full.reshape(rows, -1, BLOCK)
    with np.errstate(invalid="ignore"):
        top = np.abs(blocks).max(2, initial=0.0) if dim else np.zeros(blocks.shape[:2])
    scales = scale_bytes(top, fmt)
    bad = (scales == 255)[:, :, None]
    v = np.where(bad, 0.0, blocks) * np.exp2(127.0 - scales)[:, :, None]
    codes = nearest(v, fmt)
    half = 8 if fmt == "fp4" else 128
    codes = np.where(bad, 0, codes + half * np.signbit(np.where(bad, 0.0, blocks)))
    codes = codes.reshape(rows, -1).astype(np.uint8)
    if fmt == "fp4":
        codes = codes[:, 0::2] | codes[:, 1::2] << 4
    return codes, scales


def decode(codes: np.ndarray, scales: np.ndarray, fmt: str, dim: int) -> np.ndarray:
    """The values [rows, dim]."""
    rows = codes.shape[0]
    if fmt == "fp4":
        codes = np.stack((codes & 15, codes >> 4), 2).reshape(rows, -1)
        table = np.concatenate((grid("fp4"), -grid("fp4")))
    else:
        table = np.concatenate((grid("fp8"), [np.nan], -grid("fp8"), [np.nan]))
    scale = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (table[codes].reshape(rows, -1, BLOCK) * scale[:, :, None]).reshape(rows, -1)[:, :dim]


def unit_norm(h: np.ndarray, scale=None, eps: float = 0.0) -> np.ndarray:
    """h * scale / max(sqrt(sum h^2 + dim eps), 1e-12) per row."""
    h = h.astype(np.float64)
    with np.errstate(invalid="ignore"):
        y = h / np.maximum(np.sqrt((h * h).sum(1, keepdims=True) + h.shape[1] * eps), 1e-12)
        return y if scale is None else y * scale.astype(np.float64)


def gelu(y: np.ndarray) -> np.ndarray:
    return y * 0.5 * (1.0 + np.vectorize(math.erf, otypes=[float])(y / math.sqrt(2.0)))


def rotate(y: np.ndarray, table: np.ndarray, width: int) -> np.ndarray:
    """Columns [0, width) as queries and [width, 2 width) as keys at position row % tokens."""
    y, t = y.copy(), table.astype(np.float64)
    at = np.arange(y.shape[0]) % t.shape[1]
    for c in range(0, 2 * width, 64):
        kind = 0 if c < width else 2
        x = y[:, c:c + 64]
        swapped = x.reshape(-1, 32, 2)[:, :, ::-1].reshape(-1, 64)
        y[:, c:c + 64] = x * t[kind][at] + swapped * t[kind + 1][at]
    return y


def linear(x: np.ndarray, w: np.ndarray, bias=None, use_gelu=False, rotary=None, residual=None):
    """x [n, k] . w [k, m] (values) through the epilogue, 64 bits."""
    y = x @ w
    if bias is not None:
        y = y + bias
    if use_gelu:
        y = gelu(y)
    if rotary is not None:
        y = rotate(y, *rotary)
    return y if residual is None else y + residual.astype(np.float64)
