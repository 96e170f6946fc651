"""Microscaled rows: blocks of 32 elements of 8 or 4 bits with one power-of-two
scale each (kva_mx_*), and the norm that makes them (kva_add_rmsnorm).

They are what ``PagedKVCache.mx_project_append`` and ``mx_out_project``
multiply: weights in 4 bits, quantised and packed once,

    codes, scales = dev.empty((rows, cols // 2), np.uint8), dev.empty((rows, cols // 32), np.uint8)
    quantize(w, rows, cols, 4, codes, scales)
    packed = dev.empty(packed_bytes(rows, cols), np.uint8)
    pack_weights(codes, scales, rows, cols, packed)
    dev.synchronize()
    codes.free(), scales.free()  # a DeviceArray is held until it is freed

and activations in 8 or 4, per step.  Tensors are integer device addresses or
``DeviceArray``s (ctypes takes either); no cache is needed.  The reference has
no counterpart but its engine's own RMSNorm launches (engine.py:3043-3139).
"""
from __future__ import annotations

import ctypes

from . import _lib


def quantize(x, rows: int, cols: int, bits: int, codes, scales, x_stride: int = 0, stream=None) -> None:
    """x [rows, cols] FP16 (x_stride values between rows; 0: cols) as codes
    [rows, cols * bits / 8] and scales [rows, cols / 32]."""
    _lib.call("kva_mx_quantize", x, x_stride or cols, rows, cols, bits, codes, scales, stream)


def dequantize(codes, scales, rows: int, cols: int, bits: int, y, stream=None) -> None:
    """The values of microscaled rows, y [rows, cols] FP16."""
    _lib.call("kva_mx_dequantize", codes, scales, rows, cols, bits, y, stream)


def packed_bytes(rows: int, cols: int) -> int:
    """What pack_weights writes for a weight of rows x cols."""
    n = ctypes.c_size_t()
    _lib.call("kva_mx_packed_bytes", rows, cols, ctypes.byref(n))
    return n.value


def pack_weights(codes, scales, rows: int, cols: int, packed, stream=None) -> None:
    """4-bit weight rows in the order that the products read."""
    _lib.call("kva_mx_pack_weights", codes, scales, rows, cols, packed, stream)


def add_rmsnorm(hidden, delta, w, n_tok: int, cols: int, eps: float, out, sum_out=None, scales=None, bits: int = 16,
                stream=None) -> None:
    """sum_out = hidden + delta and out = its RMSNorm times w, as FP16 rows or
    (bits 8 or 4, with scales) microscaled ones; delta and sum_out None: the
    norm of hidden."""
    _lib.call("kva_add_rmsnorm", hidden, delta, w, n_tok, cols, eps, bits, out, scales,
              sum_out, stream)
