"""Block-scaled e4m3 in 64 bits, from its definition: the checks' side of the FP8 operators."""
from __future__ import annotations

import numpy as np

BLOCK = 128


def pitch(width):
    return -(-width // BLOCK) * BLOCK


def _table():
    v = np.empty(256)
    for b in range(256):
        e, m = (b >> 3) & 15, b & 7
        v[b] = (m / 8.0 * 2.0 ** -6 if e == 0 else (1 + m / 8.0) * 2.0 ** (e - 7)) * (-1 if b & 128 else 1)
    v[0x7f] = v[0xff] = np.nan
    return v


VALUES = _table()


def step_of(v):
    """The distance between e4m3 values around v."""
    return 2.0 ** (np.maximum(np.floor(np.log2(np.maximum(np.abs(v), 2.0 ** -9))), -6.0) - 3.0)


def nearest(v):
    """The e4m3 value nearest to v (at most 448 in size), ties to even."""
    s = step_of(v)
    return np.round(v / s) * s


def amax_of(x, block_rows):
    rows, width = x.shape
    nr, nk = -(-rows // block_rows), pitch(width) // BLOCK
    p = np.zeros((nr * block_rows, nk * BLOCK))
    p[:rows, :width] = np.abs(x)
    return np.maximum(p.reshape(nr, block_rows, nk, BLOCK).max(axis=(1, 3)), 2.0 ** -100)


def spread(scale, block_rows, rows, width):
    return np.repeat(np.repeat(scale, block_rows, 0)[:rows], BLOCK, 1)[:, :width]


def quantize(x, block_rows):
    """(e4m3 values [rows, width], scale [blocks]) of finite x, in 64 bits; and 448 x / amax."""
    x = np.asarray(x, np.float64)
    amax = amax_of(x, block_rows)
    v = x * 448.0 / spread(amax, block_rows, *x.shape)
    return nearest(v), amax / 448.0, v


def values(q, scale, block_rows, width):
    """What bytes [rows, pitch] and scales stand for, float64 [rows, width]."""
    q = np.asarray(q).view(np.uint8)
    return VALUES[q[:, :width]] * spread(np.asarray(scale, np.float64), block_rows, q.shape[0], width)


def encode(x, block_rows):
    """Bytes [rows, pitch] and float32 scales of x, as operands for a test."""
    v, scale, _ = quantize(x, block_rows)
    order = np.argsort(VALUES[:127])
    pos = VALUES[:127][order]
    idx = order[np.searchsorted(pos, np.abs(v))].astype(np.uint8)
    q = np.zeros((v.shape[0], pitch(v.shape[1])), np.uint8)
    q[:, :v.shape[1]] = idx | np.where(np.signbit(v), 128, 0).astype(np.uint8)
    return q, scale.astype(np.float32)
