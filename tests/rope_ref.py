"""Rotary positions and the norms before them in plain numpy, 64 bits, with how far a bf16 result may be off."""
from __future__ import annotations

import numpy as np

TURN = 2 * np.pi


def frequencies(rot, base, scaling=0, factor=1.0, low=1.0, high=32.0, trained=1.0):
    i = np.arange(rot // 2)
    f = base ** (-2.0 * i / max(rot, 1))
    turns = f * trained / TURN
    if scaling == 1:
        return f / factor
    if scaling == 2:
        keep = np.clip((turns - low) / (high - low), 0, 1)
    elif scaling == 3:
        at = [rot * np.log(trained / (n * TURN)) / (2 * np.log(base)) for n in (high, low)]
        lo = max(np.floor(at[0]), 0)
        hi = max(min(np.ceil(at[1]), rot - 1), lo)
        keep = np.clip((hi - i) / (hi - lo), 0, 1) if hi > lo else (i <= lo).astype(float)
    else:
        return f
    return f * keep + f / factor * (1 - keep)


def pairs(dim, first, rot, interleaved):
    """The channels (a, b) of each pair."""
    i = np.arange(rot // 2)
    return (first + 2 * i, first + 2 * i + 1) if interleaved else (first + i, first + rot // 2 + i)


def rope(x, pos, freq, first, rot, interleaved, mscale=1.0, inverse=False):
    """x [rows, heads, dim] in 64 bits rotated, and how far a kernel's bf16 result may be off.

    Bounds: the result is rounded to bf16 (half a step: 2^-8 of it, at least half of the smallest subnormal number's step,
    2^-134). The angle in turns is a product of three numbers in 64 bits (4 roundings: 2^-51 of it at most), its rest of at
    most a half may be rounded to fp32 (2^-26), times 2 pi in radians; sine and cosine are off by four steps of fp32 at most
    (2^-22), times mscale, their products with a and b and the sum another rounding each (3 x 2^-24): together less than
    2^-20 + 2 pi 2^-51 |turns| of mscale (|a| + |b|)."""
    a, b = pairs(x.shape[-1], first, rot, interleaved)
    angle = pos.astype(np.float64)[:, None, None] * np.asarray(freq, np.float64)[None, None]
    c, s = np.cos(angle) * mscale, np.sin(angle) * mscale * (-1 if inverse else 1)
    y = x.copy()
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    tol = np.zeros_like(x)
    tol[..., a] = tol[..., b] = (np.abs(x[..., a]) + np.abs(x[..., b])) * abs(mscale) * (2.0 ** -20 + 2.0 ** -51 * np.abs(angle))
    return y, tol + 2.0 ** -8 * np.abs(y) * (tol > 0) + 2.0 ** -134


def norm_rope(x, w, eps, pos, freq, first, rot, interleaved, mscale=1.0):
    """The same of x [rows, heads, dim] over each head's root mean square, times w [dim].

    Bounds: a sum of dim squares in fp32 (dim roundings, in whatever order), halved by the root; a quotient, a sum, a root,
    a reciprocal and two products, each rounded: (dim / 2 + 8) 2^-24 of every channel before the rotation."""
    dim = x.shape[-1]
    z = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    y, tol = rope(z, pos, freq, first, rot, interleaved, mscale)
    part = np.abs(z)
    a, b = pairs(dim, first, rot, interleaved)
    part[..., a] = part[..., b] = (np.abs(z[..., a]) + np.abs(z[..., b])) * abs(mscale)
    off = (dim / 2 + 8) * 2.0 ** -24
    return y, tol + 1.01 * off * part + 2.0 ** -8 * np.abs(y)
