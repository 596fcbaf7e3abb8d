"""Plain definitions of the 4-bit floating point formats (test infrastructure, numpy).

``quantize`` follows the library's definition step by step in float32 where the definition says so;
``values`` and ``tiles`` work from the bit layouts alone, in float64.
"""

from __future__ import annotations

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
BLOCK = {"nvfp4": 16, "mxfp4": 32}


def e4m3_values() -> np.ndarray:
    """float64 values of the 256 e4m3 bytes."""
    out = np.empty(256)
    for b in range(256):
        e, m = (b >> 3) & 15, b & 7
        v = m * 2.0**-9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        if e == 15 and m == 7:
            v = np.nan
        out[b] = -v if b & 128 else v
    return out


def scale_values(fmt: str) -> np.ndarray:
    if fmt == "nvfp4":
        return e4m3_values()
    out = 2.0 ** (np.arange(256, dtype=np.float64) - 127)
    out[255] = np.nan
    return out


def rotate(x: np.ndarray) -> np.ndarray:
    """The 256-wide ConvRot rotation of float32 rows in the reference's order of sums."""
    y = (x.astype(np.float32) * np.float32(0.0625)).reshape(-1, 4, 4, 4, 4)
    for axis in (4, 3, 2, 1):
        x0, x1, x2, x3 = np.moveaxis(y, axis, 0)
        t, b = x0 + x1, x0 - x1
        y = np.stack(((t + x2) - x3, (t - x2) + x3, (b + x2) + x3, (x2 - b) + x3), axis)
    return y.reshape(x.shape)


def rotation_matrix() -> np.ndarray:
    h = np.array([[1, 1, 1, -1], [1, 1, -1, 1], [1, -1, 1, 1], [-1, 1, 1, 1]]) / 2.0
    h2 = np.kron(h, h)
    return np.kron(h2, h2)


def nearest(v: np.ndarray, grid: np.ndarray) -> np.ndarray:
    """Place in `grid` of the nearest value, ties to the even place; saturating."""
    hi = np.clip(np.searchsorted(grid, v), 1, len(grid) - 1)
    lo = hi - 1
    below, above = v - grid[lo], grid[hi] - v
    up = (above < below) | ((above == below) & (hi % 2 == 0))
    return np.where(up, hi, lo)


def quantize(x: np.ndarray, fmt: str, rotation: int):
    """(codes [rows, k/2] uint8, block scale bytes [rows, k/block], row scales [rows]) of float32 rows."""
    with np.errstate(all="ignore"):
        v = rotate(x) if rotation else x.astype(np.float32)
    rows, k = v.shape
    block = BLOCK[fmt]
    bad = ~np.isfinite(v).all(1)
    v = np.where(bad[:, None], np.float32(0), v).astype(np.float32)
    blocks = v.reshape(rows, k // block, block)
    amax = np.abs(blocks).max(2)
    row = np.ones(rows, np.float32)
    if fmt == "nvfp4":
        top = amax.max(1)
        m, e = np.frexp(top / np.float32(2688))
        e = np.maximum(np.where(m > 0.5, e, e - 1), -126)
        row = np.where(top == 0, np.float32(1), np.ldexp(np.float32(1), e).astype(np.float32))
        blocks = blocks / row[:, None, None]
        want = (amax / row[:, None]) / np.float32(6)
        byte = nearest(want.astype(np.float64), e4m3_values()[:127]).astype(np.uint8)
        div = e4m3_values()[byte].astype(np.float32)
    else:
        e = np.maximum(np.where(amax == 0, -127, np.frexp(amax)[1] - 3), -127)
        byte = (e + 127).astype(np.uint8)
        div = scale_values(fmt)[byte].astype(np.float32)
    safe = np.where(div == 0, np.float32(1), div)[:, :, None]
    q = np.where(div[:, :, None] == 0, np.copysign(np.float32(0), blocks), blocks / safe).astype(np.float32)
    code = (nearest(np.abs(q).astype(np.float64), GRID) + 8 * np.signbit(q)).astype(np.uint8).reshape(rows, k)
    code[bad] = 0
    byte = np.where(bad[:, None], 0, byte).astype(np.uint8)
    return code[:, 0::2] | (code[:, 1::2] << 4), byte, np.where(bad, np.float32(np.nan), row)


def tiles(scales: np.ndarray) -> np.ndarray:
    """Plain scale bytes [rows, blocks] in tiles [rows/128, blocks/4, 32, 16], byte by byte."""
    rows, blocks = scales.shape
    out = np.zeros((-(-rows // 128), -(-blocks // 4), 32, 16), np.uint8)
    r, b = np.meshgrid(np.arange(rows), np.arange(blocks), indexing="ij")
    out[r // 128, b // 4, r % 32, 4 * (r % 128 // 32) + b % 4] = scales
    return out


def untile(t: np.ndarray, rows: int, blocks: int) -> np.ndarray:
    r, b = np.meshgrid(np.arange(rows), np.arange(blocks), indexing="ij")
    return t[r // 128, b // 4, r % 32, 4 * (r % 128 // 32) + b % 4]


def values(codes: np.ndarray, scale_bytes: np.ndarray, fmt: str) -> np.ndarray:
    """float64 values of codes times (plain) block scales."""
    rows, half = codes.shape
    c = np.empty((rows, 2 * half), np.uint8)
    c[:, 0::2], c[:, 1::2] = codes & 15, codes >> 4
    v = np.where(c & 8, -GRID[c & 7], GRID[c & 7])
    return v * np.repeat(scale_values(fmt)[scale_bytes], BLOCK[fmt], axis=1)
