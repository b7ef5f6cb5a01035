"""Rotary positions with several axes, in 64 bits (angles exact to that)."""
from __future__ import annotations

import numpy as np


def pair_axis(sections, interleaved=False):
    """Position axis of each of the 64 dimension pairs."""
    n = len(sections)
    if interleaved:
        return [i % n if i < n * sections[i % n] else 0 for i in range(64)]
    return [a for a, c in enumerate(sections) for _ in range(c)]


def rotate(x, positions, axis, inv_freq, scaling=1.0):
    """x ``[rows, heads, 128]`` float64, positions ``[A, rows]`` ints -> rotated."""
    pos = np.asarray(positions)
    y = np.array(x, dtype=np.float64)
    for i in range(64):
        # long double keeps the angle of a far position
        ang = pos[axis[i]].astype(np.longdouble) * np.longdouble(inv_freq[i])
        c = np.cos(ang).astype(np.float64)[:, None] * scaling
        s = np.sin(ang).astype(np.float64)[:, None] * scaling
        lo, hi = np.array(x[..., i], np.float64), np.array(x[..., i + 64], np.float64)
        y[..., i] = lo * c - hi * s
        y[..., i + 64] = hi * c + lo * s
    return y
