"""Microscaled blocks, the product with a 4-bit weight and the loss over a vocabulary of it, in 64 bits and
from their definitions (numpy; no code of the library)."""
from __future__ import annotations

import numpy as np

FP4 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
FP6 = np.concatenate([np.arange(8) / 8, 1 + np.arange(8) / 8, 2 + np.arange(8) / 4, 4 + np.arange(8) / 2])
TABLE, BITS = {4: FP4, 6: FP6}, {4: 4, 6: 6}


def scale_of(byte):
    return np.where(byte == 255, np.nan, np.exp2(byte.astype(np.float64) - 127))


def quantise(x, fmt):
    """Codes [rows][blocks][32] and bytes [rows][blocks] of x [rows][cols]."""
    x = np.asarray(x, np.float32)
    x = np.pad(x, ((0, 0), (0, -x.shape[1] % 32))).reshape(len(x), -1, 32)
    top = np.abs(x).max(2)
    bad = ~np.isfinite(x).all(2)
    e = np.frexp(np.where(bad, 1, top).astype(np.float64))[1] - 1
    byte = np.where(top == 0, 1, np.maximum(e - 2 + 127, 1))
    a = np.abs(np.where(bad[..., None], 0, x).astype(np.float64)) / scale_of(byte)[..., None]
    t = TABLE[fmt]
    up = np.clip(np.searchsorted(t, a), 0, len(t) - 1)
    lo = np.maximum(up - 1, 0)
    over, under = t[up] - a, a - t[lo]
    near = np.where((over < under) | ((over == under) & (up % 2 == 0)) | (a >= t[-1]), up, lo)
    codes = near | np.where(np.signbit(x), len(t), 0)
    return codes.astype(np.int64), np.where(bad, 255, byte).astype(np.uint8)


def values(codes, byte, fmt, cols):
    n = len(TABLE[fmt])
    v = TABLE[fmt][codes & (n - 1)] * np.where(codes >= n, -1.0, 1.0)
    return (v * scale_of(byte)[..., None]).reshape(len(codes), -1)[:, :cols]


def pack(codes, fmt):
    """Bytes [rows][blocks * 16 or 24] of codes, the first in the lowest bits."""
    b = BITS[fmt]
    bits = (codes[..., None] >> np.arange(b)) & 1
    return np.packbits(bits.reshape(len(codes), -1).astype(np.uint8), axis=1, bitorder="little")


def unpack(data, rows, blocks, fmt):
    b = BITS[fmt]
    bits = np.unpackbits(data.reshape(rows, -1), axis=1, bitorder="little").reshape(rows, blocks, 32, b)
    return (bits.astype(np.int64) << np.arange(b)).sum(-1)


def taken(x, act):
    """The rows as a product takes them."""
    return np.asarray(x, np.float64) if act == 32 else values(*quantise(x, act), act, x.shape[1])


def cut_error(x, act):
    """Bound of |x' - the rows as held|: 2^-23 of a block's largest value, and 2^-130 (0 where rows are quantised)."""
    if act != 32:
        return np.zeros(x.shape)
    b = np.pad(np.abs(np.asarray(x, np.float64)), ((0, 0), (0, -x.shape[1] % 32))).reshape(len(x), -1, 32).max(2)
    return np.repeat(b * 2.0 ** -23 + 2.0 ** -130, 32, 1)[:, :x.shape[1]]


def weight(rng, N, K, size=1.0, spread=0):
    """Codes and bytes of N rows of K inputs, as stored, and W [K][N] in 64 bits.  spread: binades over which the rows' sizes are drawn."""
    w = rng.normal(size=(N, K)) * size
    if spread:
        w *= np.exp2(-rng.integers(0, spread + 1, (N, 1)).astype(np.float64))
    c, b = quantise(w.astype(np.float32), 4)
    return pack(c, 4), b, values(c, b, 4, K).T


def loss(h, W, targets, act, dloss=None):
    """lse, loss and dh of rows, and the logits."""
    x = taken(h, act)
    z = x @ W
    top = z.max(1, keepdims=True)
    e = np.exp(z - top)
    total = e.sum(1, keepdims=True)
    lse = (top + np.log(total))[:, 0]
    t = np.asarray(targets)
    live = (t >= 0) & (t < W.shape[1])
    row = np.arange(len(z))
    at = np.where(live, t, 0)
    p = e / total
    p[row, at] -= 1
    g = np.where(live, 1.0 if dloss is None else np.asarray(dloss, np.float64), 0.0)
    return lse, np.where(live, lse - z[row, at], 0.0), g[:, None] * (p @ W.T) if live.any() else np.zeros(h.shape), z
