"""AdamW with fp32 or 8-bit block moments in numpy. The 8-bit forms are defined by
fp32 roundings of the averages and by the values of the codes; here they are
reached over float64 arithmetic on values, not over bit patterns."""

from __future__ import annotations

import numpy as np

BLOCK = 128


def mix(x: np.ndarray) -> np.ndarray:
    x = np.asarray(x, dtype=np.uint32)
    with np.errstate(over="ignore"):
        x = (x ^ (x >> np.uint32(16))) * np.uint32(0x9E3779B9)
        x = (x ^ (x >> np.uint32(15))) * np.uint32(0xBB67AE85)
    return x ^ (x >> np.uint32(16))


def noise(n: int, seed: int, step: int, group: int, at: int = 0):
    """(m's, v's) 16 random bits of positions at .. at + n - 1."""
    pos = at + np.arange(n, dtype=np.int64)
    high = (pos >> 32).astype(np.uint32)
    u = np.uint32
    with np.errstate(over="ignore"):
        key = mix(mix(u(seed)) + u(step))
        if group:
            key = mix(key + u(group))
        key = np.where(high != 0, mix(key + high), key)
        h = mix((pos & 0xFFFFFFFF).astype(np.uint32) + key)
    return h & u(0xFFFF), h >> u(16)


def block_exponents(x: np.ndarray) -> np.ndarray:
    """Stored exponents of flat x (padded to blocks with zeros)."""
    v = np.zeros(-(-x.size // BLOCK) * BLOCK, dtype=np.float64)
    v[:x.size] = x.reshape(-1)
    v = v.reshape(-1, BLOCK)
    bad = ~np.isfinite(v).all(-1)
    amax = np.where(bad, 1.0, np.abs(np.where(np.isfinite(v), v, 0)).max(-1))
    _, e = np.frexp(amax)
    e = np.where(amax == 0, -126, np.clip(e - 1, -126, 126))
    return np.where(bad, 255, e + 127).astype(np.uint8)


def level_table(ebits: int) -> np.ndarray:
    """The magnitudes of the codes, ascending."""
    low = 2 - (1 << ebits)
    c = np.arange(8 << ebits)
    e, f = c >> 3, (c & 7).astype(np.float64)
    return np.where(e == 0, np.ldexp(f / 8, low), np.ldexp(1 + f / 8, np.maximum(e - 1, 0) + low))


def encode(x: np.ndarray, ebits: int, signed: bool, bits16: np.ndarray):
    """fp32 flat x, 16 random bits each -> (codes, exponents)."""
    x = np.asarray(x, dtype=np.float32).reshape(-1)
    exps = block_exponents(x)
    e = np.repeat(exps.astype(np.int64), BLOCK)[:x.size]
    fine = np.where(np.isfinite(x), x, 0).astype(np.float64)
    y = np.ldexp(np.abs(fine), 127 - e)
    low = 2.0 ** (2 - (1 << ebits))
    # Below the smallest full binade y is first rounded to 24 bits of y + low.
    y = np.where(y < low, (y + low).astype(np.float32).astype(np.float64) - low, y)
    levels = level_table(ebits)
    i = np.searchsorted(levels, y, side="right") - 1
    step = np.where(i + 1 < levels.size, levels[np.minimum(i + 1, levels.size - 1)] - levels[i], 1.0)
    up = np.floor((y - levels[i]) / step + bits16.astype(np.float64) / 65536)
    code = np.minimum(i + up, levels.size - 1).astype(np.int64)
    if signed:
        code = code + 128 * np.signbit(x)
    return np.where(e == 255, 0, code).astype(np.uint8), exps


def decode(codes: np.ndarray, exps: np.ndarray, ebits: int, signed: bool) -> np.ndarray:
    c = codes.reshape(-1).astype(np.int64)
    mag = c & 127 if signed else c
    e = np.repeat(exps.astype(np.int64), BLOCK)[:c.size]
    y = np.ldexp(level_table(ebits)[mag], e - 127)
    y = np.where(signed & (c >= 128), -y, y)
    return np.where(e == 255, np.nan, y)


def averages(g, m, v, beta1: float, beta2: float):
    """m', v' with every operation rounded to fp32."""
    f = np.float32
    g, m, v = (np.asarray(t, dtype=np.float32) for t in (g, m, v))
    with np.errstate(over="ignore", invalid="ignore"):
        return (m * f(beta1) + g * f(1 - beta1)).astype(f), (v * f(beta2) + (g * f(1 - beta2)) * g).astype(f)


def update(p, m, v, *, lr, beta1, beta2, eps, weight_decay, step):
    """float64 p' from the new averages."""
    p, m, v = (np.asarray(t, dtype=np.float64) for t in (p, m, v))
    denom = np.sqrt(v) / np.sqrt(1 - beta2 ** step) + eps
    with np.errstate(divide="ignore", invalid="ignore"):
        return p * (1 - lr * weight_decay) - lr / (1 - beta1 ** step) * (m / denom)
