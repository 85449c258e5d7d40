"""The 4-bit paged cache's operators written out plainly: rows and codes from the definitions, in numpy."""
from __future__ import annotations

import numpy as np

import kv8_plain
from aihost_b200 import ROPE_INTERLEAVED, ROPE_NONE

TINY = np.float32(2.0 ** -24)


def rotate32(x, pos, theta, mode):
    """x [n, heads, d] fp32 rotated at pos [n]: angles in fp32, cosines and sines of those rounded once, products and sums
    in fp32."""
    if mode == ROPE_NONE:
        return x
    d = x.shape[-1]
    ang = (np.asarray(pos, dtype=np.float32)[:, None] * kv8_plain.freqs(theta, d)).astype(np.float64)[:, None, :]
    c, s = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    out = np.array(x)
    i, j = (np.s_[..., 0::2], np.s_[..., 1::2]) if mode == ROPE_INTERLEAVED else (np.s_[..., :d // 2], np.s_[..., d // 2:])
    out[i], out[j] = x[i] * c - x[j] * s, x[i] * s + x[j] * c
    return out


def quantise(x):
    """(codes [..., d] uint8, low [...], step [...] fp16) of fp32 rows x [..., d]."""
    with np.errstate(all="ignore"):
        low = x.min(-1).astype(np.float16)
        low32 = low.astype(np.float32)
        step = ((x.max(-1) - low32) * np.float32(1 / 15)).astype(np.float16)
        step = np.maximum(step, np.float16(TINY))
        bad = ~(np.isfinite(x).all(-1) & np.isfinite(low) & np.isfinite(step))
        inv = np.float32(1) / step.astype(np.float32)
        y = np.rint((x - low32[..., None]) * inv[..., None]).clip(0, 15)
    y[bad] = 0
    low[bad] = step[bad] = np.nan
    return y.astype(np.uint8), low, step


def pack(codes):
    """Codes [..., d] as bytes [..., d / 2]: of eight elements the nibbles e0 e2, e4 e6, e1 e3, e5 e7."""
    c = codes.reshape(*codes.shape[:-1], -1, 8)
    return np.stack([c[..., a] | c[..., b] << 4 for a, b in ((0, 2), (4, 6), (1, 3), (5, 7))], -1).reshape(*codes.shape[:-1], -1)


def unpack(pool):
    b = pool.reshape(*pool.shape[:-1], -1, 4)
    out = np.empty(b.shape[:-1] + (8,), np.uint8)
    for k, (lo, hi) in enumerate(((0, 2), (4, 6), (1, 3), (5, 7))):
        out[..., lo], out[..., hi] = b[..., k] & 15, b[..., k] >> 4
    return out.reshape(*pool.shape[:-1], -1)


def values(pool, rng, dtype=np.float32):
    """What codes [..., d / 2] with ranges [..., 2] stand for: low + step * code, rounded to dtype once."""
    r = rng.astype(np.float64)
    with np.errstate(invalid="ignore"):
        return (r[..., :1] + r[..., 1:] * unpack(pool).astype(np.float64)).astype(dtype)
