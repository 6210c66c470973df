"""CPU oracle of the 4-bit key/value cache operators (test infrastructure).

Restates the definitions in NumPy: the rotation and the 4-bit quantizer in
fp32 with one rounding per operation (their results are compared bit for
bit), attention in fp64.
"""
from __future__ import annotations

import numpy as np

__all__ = ["bf16", "rotate", "quantise", "values", "pack", "unpack", "attention"]


def bf16(x):
    """fp32 rounded to bf16 (nearest even), as fp32; NaN and Inf kept."""
    x = np.asarray(x, np.float32)
    b = x.view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)
    return np.where(np.isfinite(x), r, x).astype(np.float32)


def rotate(x, table, positions, interleaved=False, inverse=False):
    """x [T, H, D] fp32; each product and each sum rounded to fp32."""
    x = np.asarray(x, np.float32)
    half = table.shape[1] // 2
    t = table[positions][:, None]
    c, s = t[..., :half], t[..., half:]
    if inverse:
        s = -s
    y = x.copy()
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
    else:
        a, b = x[..., :half], x[..., half:2 * half]
    with np.errstate(all="ignore"):
        ya, yb = a * c - b * s, b * c + a * s
    if interleaved:
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = ya, yb
    else:
        y[..., :half], y[..., half:2 * half] = ya, yb
    return y


def quantise(x, group):
    """(codes int8 [..., D], scales fp16 [..., D / group]) of finite fp32 x."""
    parts = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, group)
    with np.errstate(over="ignore"):
        s = bf16(np.abs(parts).max(-1) / np.float32(7)).astype(np.float16)
    s = np.minimum(s, np.float16(9344))
    s = np.where(s == 0, np.float16(1), s).astype(np.float16)
    with np.errstate(over="ignore"):
        q = np.clip(np.rint(parts / s.astype(np.float32)[..., None]), -7, 7).astype(np.int8)
    return q.reshape(x.shape), s


def pack(codes):
    low, high = codes[..., 0::2] & 15, codes[..., 1::2] & 15
    return (low | (high << 4)).astype(np.uint8)


def unpack(packed):
    n = np.stack([packed & 15, packed >> 4], -1).reshape(*packed.shape[:-1], -1).astype(np.int8)
    return np.where(n > 7, n - 16, n).astype(np.int8)


def values(codes, scales):
    """fp64 code * scale."""
    g = codes.shape[-1] // scales.shape[-1]
    with np.errstate(invalid="ignore"):
        return codes.astype(np.float64) * np.repeat(scales.astype(np.float64), g, -1)


def attention(q, k, v, scale, count, window=0, causal=True):
    """One sequence in fp64: q [count, Hq, D], the sequence's cached k, v [n,
    Hk, D].  Returns (out, log_sum, spread, size, mass): spread = sum p |v| per
    output, size [count, Hq] = the largest scale * sum |q| |k| a row sees,
    mass = sum |v| per output -- what the errors of the weights (relative), of
    the scores and of the weights (absolute) are bounded by."""
    n, heads, kv = k.shape[0], q.shape[1], k.shape[1]
    out = np.zeros(q.shape)
    spread, mass = np.zeros(q.shape), np.zeros(q.shape)
    lse = np.full(q.shape[:2], -np.inf)
    size = np.zeros(q.shape[:2])
    for i in range(count):
        p = n - count + i
        hi = min(p + 1, n) if causal else n
        lo = max(0, p + 1 - window) if window else 0
        if hi <= lo or hi <= 0:
            continue
        for h in range(heads):
            kk, vv = k[lo:hi, h * kv // heads], v[lo:hi, h * kv // heads]
            s = scale * (kk @ q[i, h].astype(np.float64))
            m = s.max()
            e = np.exp(s - m)
            out[i, h] = (e @ vv) / e.sum()
            spread[i, h] = (e @ np.abs(vv)) / e.sum()
            mass[i, h] = np.abs(vv).sum(0)
            lse[i, h] = m + np.log(e.sum())
            size[i, h] = abs(scale) * (np.abs(kk) @ np.abs(q[i, h].astype(np.float64))).max()
    return out, lse, spread, size, mass
