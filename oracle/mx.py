"""The block-scaled cache in numpy and 64 bits (TEST INFRASTRUCTURE ONLY; the product never imports it).

Blocks of 32 numbers as ``include/diffcache_hip.h`` defines them (``dc_mx_store``), and softmax attention over them.  The
reference has no such cache: PARITY UNPINNED there, pinned by the format's definition.
"""
from __future__ import annotations

import numpy as np

EMAX = {4: 2, 8: 8}
LAST = {4: 7, 8: 126}                 # code of the largest number
LIMITS = {4: (2, 252), 8: (10, 246)}


def grid(bits: int) -> np.ndarray:
    """The number of every code, sign bit included."""
    half = 1 << (bits - 1)
    m_bits, bias = (1, 1) if bits == 4 else (3, 7)
    out = np.empty(2 * half)
    for c in range(half):
        e, m = c >> m_bits, c & ((1 << m_bits) - 1)
        out[c] = np.ldexp(m, 1 - bias - m_bits) if e == 0 else np.ldexp(m + (1 << m_bits), e - bias - m_bits)
    if bits == 8:
        out[127] = np.nan
    out[half:] = -out[:half]
    return out


def _nearest(a: np.ndarray, bits: int) -> np.ndarray:
    """Codes of non-negative numbers, rounded to nearest with ties to the even code; len(grid) / 2 - 1 and beyond past the end."""
    g = grid(bits)[:LAST[bits] + 1]
    step = g[-1] - g[-2]
    g = np.append(g, g[-1] + step)                       # where the next number would be
    up = np.minimum(np.searchsorted(g, np.minimum(a, g[-1])), len(g) - 1)
    down = np.maximum(up - 1, 0)
    du, dd = g[up] - a, a - g[down]
    return np.where(du < dd, up, np.where(du > dd, down, np.where(up % 2 == 0, up, down)))


def encode(x: np.ndarray, bits: int):
    """x (..., hd) -> codes (..., hd * bits / 8), scale (..., hd / 32), both uint8.  The scale is the least exponent at which the
    block's largest number does not round past the last code, found by trying."""
    x = np.asarray(x, dtype=np.float64)
    blocks = x.reshape(-1, 32)
    lo, hi = LIMITS[bits]
    with np.errstate(over="ignore", invalid="ignore"):
        most = np.max(np.abs(blocks), axis=1)
    fine = np.isfinite(most)
    safe = np.where(fine, most, 0.0)
    # (one less than what brings the largest number's leading bit to the last code's never fits: try that one, then one more)
    first = np.frexp(safe)[1] - 1 - EMAX[bits] + 127
    fits = _nearest(np.ldexp(safe, 127 - first), bits) <= LAST[bits]
    e = np.where(safe > 0, np.where(fits, first, first + 1), lo)
    e = np.clip(e, lo, hi)
    y = np.where(fine[:, None], blocks, 0.0) * np.ldexp(1.0, 127 - e)[:, None]
    code = np.minimum(_nearest(np.abs(y), bits), LAST[bits]) | (np.signbit(y).astype(int) << (bits - 1))
    code = code.astype(np.uint8).reshape(x.shape)
    if bits == 4:
        code = code[..., ::2] | (code[..., 1::2] << 4)
    scale = np.where(fine, e, 255).astype(np.uint8).reshape(x.shape[:-1] + (x.shape[-1] // 32,))
    return code, scale


def decode(codes: np.ndarray, scale: np.ndarray) -> np.ndarray:
    """The numbers held, (..., hd) float64; the bits follow from the shapes."""
    bits = codes.shape[-1] * 8 // (scale.shape[-1] * 32)
    if bits == 4:
        codes = np.stack([codes & 15, codes >> 4], axis=-1).reshape(codes.shape[:-1] + (-1,))
    f = np.where(scale == 255, np.nan, np.ldexp(1.0, scale.astype(int) - 127))
    return grid(bits)[codes] * np.repeat(f, 32, axis=-1)


def attended(total: int, n_sink: int = 0, window: int = 0) -> np.ndarray:
    rows = np.arange(total)
    return rows[(rows < n_sink) | (rows >= total - window)] if window else rows


def attention(q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float):
    """q (heads, hd), k and v (rows, hd): out, lse, and per head the sum of p |v| and the largest sum of |q k scale|, by which
    errors are bounded."""
    if len(k) == 0:
        z = np.zeros_like(q)
        return z, np.full(len(q), -np.inf), z, np.zeros(len(q))
    x = q @ k.T * scale
    m = x.max(1, keepdims=True)
    p = np.exp(x - m)
    total = p.sum(1, keepdims=True)
    return (p @ v) / total, (m + np.log(total))[:, 0], (p @ np.abs(v)) / total, (np.abs(q) @ np.abs(k).T * abs(scale)).max(1)
