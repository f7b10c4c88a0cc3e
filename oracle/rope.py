"""Rotary positions of several axes in numpy float64 (test infrastructure), one pair of channels after another."""

from __future__ import annotations

import numpy as np


def rotate(x: np.ndarray, pos: np.ndarray, inv_freq, axis, pairs: str, scale: float = 1.0) -> np.ndarray:
    """x [n, heads, d], pos [axes, n] -> float64 [n, heads, d]."""
    y = np.array(x, np.float64)
    half = len(inv_freq)
    for p, (f, a) in enumerate(zip(inv_freq, axis)):
        t = pos[a].astype(np.longdouble) * np.longdouble(f)  # positions of 31 bits times a double
        c, s = np.cos(t).astype(np.float64)[:, None] * scale, np.sin(t).astype(np.float64)[:, None] * scale
        i, j = (p, p + half) if pairs == "halves" else (2 * p, 2 * p + 1)
        x0, x1 = np.asarray(x[..., i], np.float64), np.asarray(x[..., j], np.float64)
        y[..., i], y[..., j] = x0 * c - x1 * s, x0 * s + x1 * c
    return y
