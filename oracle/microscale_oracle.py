"""Microscaled rows, the norm that makes them and products of them, restated in
numpy in 64 bits: what the kva_mx_* entry points and kva_add_rmsnorm are
tested against.  No counterpart in the reference.

An element is taken as the nearest of the listed values, so the lists are the
definition; nothing here rounds by arithmetic on exponents.
"""
from __future__ import annotations

import numpy as np

BLOCK = 32
#: The magnitudes of an element, by code.
GRID = {4: np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]),
        8: np.array([m / 512 for m in range(8)] +
                    [(8 + m) / 8 * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1])}
NAN_SCALE = 255


def scale_bytes(x, bits: int) -> np.ndarray:
    """x [rows, cols] in 64 bits: the scale byte of each block, [rows, cols / 32]."""
    x = np.asarray(x, np.float64)
    most = np.abs(x.reshape(x.shape[0], -1, BLOCK)).max(-1)
    units = 2.0 ** np.arange(-126, 128)
    covers = GRID[bits][-1] * units  # ascending: the first that is not below `most`
    byte = np.searchsorted(covers, np.where(np.isfinite(most), most, 0.0)) + 1
    return np.where(np.isfinite(most), byte, NAN_SCALE).astype(np.uint8)


def encode(x, bits: int):
    """x [rows, cols] as element codes [rows, cols] (unpacked) and scale bytes."""
    x = np.asarray(x, np.float64)
    b = scale_bytes(x, bits)
    bad = np.repeat(b == NAN_SCALE, BLOCK, axis=1)
    y = np.where(bad, 0.0, x) / 2.0 ** (np.repeat(np.where(b == NAN_SCALE, 127, b), BLOCK, axis=1).astype(float) - 127)
    grid, mag = GRID[bits], np.abs(y)
    hi = np.minimum(np.searchsorted(grid, mag), len(grid) - 1)
    lo = np.maximum(hi - 1, 0)
    up, down = grid[hi] - mag, mag - grid[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = np.where(np.signbit(y) & ~bad, code + (1 << (bits - 1)), code)
    return code.astype(np.uint8), b


def pack_codes(code, bits: int) -> np.ndarray:
    """Element codes as bytes: of two 4-bit ones the even in the low half."""
    return code if bits == 8 else (code[:, ::2] | code[:, 1::2] << 4).astype(np.uint8)


def unpack_codes(codes, bits: int) -> np.ndarray:
    return codes if bits == 8 else np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1)


def decode(codes, scales, bits: int) -> np.ndarray:
    """The values of packed codes and scale bytes, in 64 bits (8-bit codes 0x7f
    and 0xff and scale byte 255 are NaN)."""
    c = unpack_codes(codes, bits).astype(int)
    mag = c & ((1 << (bits - 1)) - 1)
    grid = np.append(GRID[bits], np.nan)  # 8 bits: one code more than values
    v = np.where(c >> (bits - 1) == 1, -1.0, 1.0) * grid[mag]
    s = np.where(scales == NAN_SCALE, np.nan, 2.0 ** (scales.astype(float) - 127))
    return v * np.repeat(s, BLOCK, axis=1)


def quantized(x, bits: int) -> np.ndarray:
    """The values that microscaled rows of x have."""
    code, b = encode(x, bits)
    return decode(pack_codes(code, bits), b, bits)


def pack_weights(codes, scales) -> np.ndarray:
    """4-bit rows in the order that the products read: [row tiles][cols / 64][64
    lanes][16] codes, then [row tiles][cols / 256][64 lanes][4] scales; lane l
    has row l % 32 of its tile and block l / 32 of each 64 values."""
    rows, cols = codes.shape[0], 2 * codes.shape[1]
    n = -(-rows // 32) * 32
    c, s = np.zeros((n, cols // 2), np.uint8), np.ones((n, cols // BLOCK), np.uint8)
    c[:rows], s[:rows] = codes, scales
    c = c.reshape(n // 32, 32, cols // 64, 2, 16).transpose(0, 2, 3, 1, 4)
    s = s.reshape(n // 32, 32, cols // 256, 4, 2).transpose(0, 2, 4, 1, 3)
    return np.concatenate([c.reshape(-1), s.reshape(-1)])


def add_rmsnorm(hidden, delta, w, eps: float):
    """(fp16 sums, their norm times w in 64 bits)."""
    total = np.asarray(hidden, np.float16)
    if delta is not None:
        total = (total.astype(np.float64) + np.asarray(delta, np.float64)).astype(np.float16)
    x = total.astype(np.float64)
    return total, x / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps) * np.asarray(w, np.float64)
