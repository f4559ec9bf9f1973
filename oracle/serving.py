"""CPU oracle of the serving operators: paged append with rotation, attention over the paged cache,
int8 linear layers.  TEST INFRASTRUCTURE ONLY, like ``oracle.py`` beside it.

The reference has no operator file for these; the functions restate the definitions of
``include/b200ops.h`` in numpy float64, and ``tests/test_serving_oracle.py`` holds them to
properties and small cases worked out by hand.  16-bit arrays are float64 arrays of values the
type holds.
"""
from __future__ import annotations

import numpy as np

# digits of a value, exponent (as of frexp) below which the steps stop shrinking
_FORMAT = {"bfloat16": (8, -125), "float16": (11, -13), "float32": (24, -125)}


def nearest(x, dtype):
    """float64 values rounded once to the nearest value of ``dtype``, ties to even (float64).
    Infinities and NaN stay; nothing here overflows."""
    x = np.asarray(x, dtype=np.float64)
    digits, lowest = _FORMAT[dtype]
    with np.errstate(invalid="ignore"):
        _, exponent = np.frexp(np.where(np.isfinite(x), x, 0.0))
        step = np.ldexp(1.0, np.maximum(exponent, lowest) - digits)
        return np.where(np.isfinite(x), np.rint(x / step) * step, x)


def half_step(dtype):
    """Largest relative error of one rounding to ``dtype``."""
    return 2.0 ** -_FORMAT[dtype][0]


def rotate(x, cos, sin, interleaved=False):
    """x [T, heads, D] with cos, sin [T, R / 2] of each token's position: pairs (i, i + R/2) or
    (2i, 2i + 1) become (a cos - b sin, b cos + a sin)."""
    x = np.array(x, dtype=np.float64)
    half = cos.shape[-1]
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    a, b = x[..., first].copy(), x[..., second].copy()
    c, s = np.asarray(cos, np.float64)[:, None], np.asarray(sin, np.float64)[:, None]
    x[..., first], x[..., second] = a * c - b * s, b * c + a * s
    return x


def four_bits(rows, dtype):
    """(codes, scale, low) of rows [..., D] whose values ``dtype`` holds."""
    rows = np.asarray(rows, dtype=np.float64)
    low = rows.min(-1)
    scale = nearest((rows.max(-1) - low) / 15.0, dtype)
    with np.errstate(divide="ignore", invalid="ignore"):
        codes = np.rint((rows - low[..., None]) / scale[..., None])
    codes = np.where(scale[..., None] > 0, np.clip(codes, 0, 15), 0)
    return codes.astype(np.uint8), scale, low


def stands_for(codes, scale, low):
    return low[..., None] + codes.astype(np.float64) * scale[..., None]


def pack(codes):
    """4-bit codes [..., D] -> bytes [..., D / 2], even elements in the low half."""
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).astype(np.uint8)


def unpack(packed):
    out = np.empty(packed.shape[:-1] + (packed.shape[-1] * 2,), dtype=np.uint8)
    out[..., 0::2], out[..., 1::2] = packed & 15, packed >> 4
    return out


def gather(cache, table_row, length, block):
    """Rows of one sequence, [length, heads, ...], from a cache [pages, heads, block, ...]."""
    where = np.arange(length)
    return cache[table_row[where // block], :, where % block]


def attention_rows(q, keys, values, scale, causal):
    """One sequence: q [n, H, D] against keys / values [length, H_KV, D] -> (out, lse, mass, top):
    ``mass`` = sum_j p_j |v_j| per element and ``top`` = the largest scale * sum |q_d k_jd| of each row,
    which the error bounds of the tests are built from."""
    q, keys, values = (np.asarray(t, dtype=np.float64) for t in (q, keys, values))
    n, heads, dim = q.shape
    length, group = keys.shape[0], heads // keys.shape[1]
    out, mass = np.zeros((n, heads, dim)), np.zeros((n, heads, dim))
    lse, top = np.full((n, heads), np.inf), np.zeros((n, heads))
    for i in range(n):
        seen = max(0, min(length, length - n + i + 1)) if causal else length
        if seen == 0:
            continue
        for h in range(heads):
            k, v = keys[:seen, h // group], values[:seen, h // group]
            s = scale * (k @ q[i, h])
            m = s.max()
            p = np.exp(s - m)
            lse[i, h] = m + np.log(p.sum())
            p /= p.sum()
            out[i, h], mass[i, h] = p @ v, p @ np.abs(v)
            top[i, h] = (scale * (np.abs(k) @ np.abs(q[i, h]))).max()
    return out, lse, mass, top


def quantize_rows(x):
    """(codes, scale): scale = max |x| / 127 in float32, codes = x / scale to nearest even."""
    x = np.asarray(x, dtype=np.float64)
    scale = (np.abs(x).max(-1).astype(np.float32) / np.float32(127.0)).astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        codes = np.rint(x / scale.astype(np.float64)[:, None])
    return np.where(scale[:, None] > 0, np.clip(codes, -127, 127), 0).astype(np.int8), scale
