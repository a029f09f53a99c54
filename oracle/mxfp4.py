"""MXFP4 in numpy, from the format's definition (OCP Microscaling Formats 1.0):
the arithmetic is on exact float64 values, apart from the kernels' bit forms."""

from __future__ import annotations

import numpy as np

BLOCK = 32
LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(x: np.ndarray):
    """float array [..., cols] -> (codes [..., 16 B], scales [..., B]) uint8."""
    x = np.asarray(x, dtype=np.float64)
    cols = x.shape[-1]
    blocks = -(-cols // BLOCK)
    pad = np.zeros((*x.shape[:-1], blocks * BLOCK))
    pad[..., :cols] = x
    v = pad.reshape(*x.shape[:-1], blocks, BLOCK)
    bad = ~np.isfinite(v).all(-1)
    mag = np.where(bad[..., None], 0.0, np.abs(v))
    amax = mag.max(-1)
    _, e = np.frexp(amax)  # amax = f 2^e with f in [1/2, 1)
    e = np.where(amax == 0, -127, np.clip(e - 1 - 2, -127, 125))
    y = np.ldexp(mag, -e[..., None])
    # Distance to each level; of two nearest the one of even code.
    d = np.abs(y[..., None] - LEVELS)
    best = d.min(-1, keepdims=True)
    near = d == best
    first = near.argmax(-1)
    last = 7 - near[..., ::-1].argmax(-1)
    code = np.where(first % 2 == 0, first, last)
    code = np.where(bad[..., None], 0, code + 8 * np.signbit(v))
    code = code.reshape(*x.shape[:-1], blocks * BLOCK).astype(np.uint8)
    packed = code[..., 0::2] | (code[..., 1::2] << 4)
    return packed, np.where(bad, 255, e + 127).astype(np.uint8)


def dequantize(codes: np.ndarray, scales: np.ndarray, cols: int) -> np.ndarray:
    """float64 [..., cols]."""
    c = np.stack([codes & 15, codes >> 4], axis=-1).reshape(*codes.shape[:-1], -1)
    v = LEVELS[c & 7] * np.where(c & 8, -1.0, 1.0)
    e = np.repeat(scales.astype(np.int64), BLOCK, axis=-1)
    out = np.where(e == 255, np.nan, np.ldexp(v, e - 127))
    return out[..., :cols]


def roundtrip(x: np.ndarray) -> np.ndarray:
    return dequantize(*quantize(x), np.asarray(x).shape[-1])
