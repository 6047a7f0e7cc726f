"""Rotary positions from their definition, with the bound that the kernel's arithmetic allows.

Angles: position times frequency (64-bit numbers) in extended precision, modulo a turn; sine, cosine and the rest in 64
bits.  For a pair (a, b) after the norm, with r = scale (|a| + |b|), the error of one output y is at most

  u |y|             rounding to the result's type, u half a step (2^-8, 2^-11, 2^-24), or 2^-25 below float16's normal range;
  8 2^-24 r         the angle within an eighth of a turn: its conversion, its factor 2 pi 2^-32 (pi / 4 2^-24 each) and its
                    truncation (2 pi 2^-32), the polynomials' last operations (2^-24) and remainders (2^-28): below
                    4 2^-24 of each sine and cosine; the factor, the product, the other product and their sum: 2^-24 each;
  (dim / 2 + 12) 2^-24 r   with a norm: the sum of dim squares (relative dim 2^-24 at most, half of that in the root),
                    the mean, eps, the root to two steps, and two products.
"""
from __future__ import annotations

import numpy as np
import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def angles(radians, positions):
    """Angles modulo a turn [tokens][pairs] as float64."""
    turn = np.longdouble("6.283185307179586476925286766559005768")
    p = np.asarray(positions, dtype=np.int64).astype(np.longdouble)[:, None]
    share = np.asarray(radians, dtype=np.float64).astype(np.longdouble)[None] / turn * p
    share -= np.floor(share)
    return torch.from_numpy((share * turn).astype(np.float64))


def rotate(x, positions, radians, scale, layout, norm=None, eps=1e-6, inverse=False, dtype=None):
    """x [tokens][heads][dim] on the CPU -> (y, bound) in 64 bits for results of `dtype`."""
    u = UNIT[dtype or x.dtype]
    dim, n = x.shape[-1], 2 * len(radians)
    x = x.double()
    share = 8.0
    if norm is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * norm.double()
        share += dim / 2 + 12
    angle = angles(radians, positions)
    c, s = torch.cos(angle)[:, None] * scale, torch.sin(angle)[:, None] * scale
    if inverse:
        s = -s
    y, r = x.clone(), torch.zeros_like(x)
    ia, ib = (slice(0, n // 2), slice(n // 2, n)) if layout == "half" else (slice(0, n, 2), slice(1, n, 2))
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    r[..., ia] = r[..., ib] = abs(scale) * (a.abs() + b.abs())
    r[..., n:] = x[..., n:].abs() if norm is not None else 0.0
    tiny = 2.0 ** -25 if u == 2.0 ** -11 else 0.0
    return y, u * y.abs() + share * 2.0 ** -24 * r * (1 + 2 * u) + tiny + 1e-30
