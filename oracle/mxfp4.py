"""Microscaled 4-bit matrices restated in 64-bit numpy from the definition: the test oracle of the MXFP4 entry points.

A block of 32 consecutive elements of a row shares 2^e, e = floor(log2(max |x|)) - 2 (at least -127), and holds e2m1
numbers: sign and one of GRID, nearest with ties to the even code, at most 6.  A block with an infinity or NaN is NaN.
"""
from __future__ import annotations

import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
NAN = 255


def blocks(cols: int) -> int:
    return -(-cols // 32)


def quantize(x):
    """(codes [rows][16 * blocks], scale bytes [rows][blocks]) of a real matrix."""
    x = np.asarray(x, dtype=np.float64)
    rows, cols = x.shape
    full = np.zeros((rows, blocks(cols) * 32))
    full[:, :cols] = x
    full = full.reshape(rows, -1, 32)
    most = np.abs(full).max(axis=2)
    bad = ~np.isfinite(full).all(axis=2)
    _, e = np.frexp(np.where(bad | (most == 0), 1.0, most))   # most = f * 2^e, 0.5 <= f < 1: floor(log2) = e - 1
    e = np.where(most == 0, -127, np.maximum(e - 3, -127))
    y = np.abs(np.where(bad[..., None], 0.0, full)) * np.exp2(-e.astype(np.float64))[..., None]
    code = np.zeros(y.shape, dtype=np.uint8)
    for i in range(7):   # a border itself goes to the even code beside it
        border = (GRID[i] + GRID[i + 1]) / 2
        code += (y > border) | ((y == border) & (i % 2 == 1))
    code = np.where(bad[..., None], 0, code | (np.signbit(full).astype(np.uint8) << 3)).astype(np.uint8)
    code = code.reshape(rows, -1, 2)
    return code[..., 0] | (code[..., 1] << 4), np.where(bad, NAN, e + 127).astype(np.uint8)


def tile_scales(s):
    """Scale bytes [rows][blocks] in the order they are kept: tiles of 128 rows x 4 blocks, zeros where nothing is."""
    rows, nb = s.shape
    high, wide = -(-rows // 128), -(-nb // 4)
    out = np.zeros(high * wide * 512, dtype=np.uint8)
    r, b = np.meshgrid(np.arange(rows), np.arange(nb), indexing="ij")
    out[((r // 128) * wide + b // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4] = s
    return out


def untile_scales(t, rows, cols):
    nb = blocks(cols)
    wide = -(-nb // 4)
    r, b = np.meshgrid(np.arange(rows), np.arange(nb), indexing="ij")
    return np.asarray(t)[((r // 128) * wide + b // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4]


def values(codes, scales, cols):
    """Real values of codes [rows][16 * blocks] with scale bytes [rows][blocks]."""
    codes = np.asarray(codes)
    c = np.stack([codes & 15, codes >> 4], axis=2).reshape(codes.shape[0], -1, 32)
    v = np.where(c & 8, -1.0, 1.0) * GRID[c & 7]
    s = np.where(scales == NAN, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (v * s[..., None]).reshape(codes.shape[0], -1)[:, :cols]


def rounded(x):
    """The values that quantisation leaves of x."""
    codes, scales = quantize(x)
    return values(codes, scales, np.asarray(x).shape[1])
