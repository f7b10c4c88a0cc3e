"""MXFP4 weights restated in numpy float64 (test infrastructure): the e2m1 code table, the quantizer, the gated block.  No function
of the reference covers them."""

from __future__ import annotations

import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
EMIN, EMAX = -23, 13


def values(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """codes uint8 [n, k / 2] (even column in the lower nibble), scales uint8 [n, ceil(k / 32)] -> float64 [n, k]."""
    n, half = codes.shape
    nib = np.stack([codes & 15, codes >> 4], -1).reshape(n, 2 * half)
    v = E2M1[nib & 7] * np.where(nib & 8, -1.0, 1.0)
    return v * np.exp2(np.repeat(scales.astype(np.float64) - 127, 32, axis=1)[:, :2 * half])


def exponent(top: np.ndarray) -> np.ndarray:
    """The smallest e in [EMIN, EMAX] with top <= 6 * 2^e; 0 for zero groups."""
    top = np.asarray(top, np.float64)
    e = np.full(top.shape, EMIN)
    for x in range(EMIN + 1, EMAX + 1):
        e = np.where(top > 6 * 2.0 ** (x - 1), x, e)
    return np.where(top == 0, 0, e)


def quantize(w: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """w [n, k] -> (codes, scales): nearest code, ties to the even one."""
    n, k = w.shape
    g = -(-k // 32)
    p = np.zeros((n, g * 32))
    p[:, :k] = w
    e = exponent(np.abs(p.reshape(n, g, 32)).max(-1))
    x = np.abs(p) / np.exp2(np.repeat(e, 32, axis=1))
    d = np.abs(x[..., None] - E2M1)
    near = d.min(-1, keepdims=True)
    pick = np.where((d == near) & (np.arange(8) % 2 == 0), 2, (d == near).astype(int)).argmax(-1)  # of two equally near codes the even one
    c = (pick | np.where(np.signbit(p), 8, 0)).astype(np.uint8)[:, :k]
    return c[:, 0::2] | (c[:, 1::2] << 4), (e + 127).astype(np.uint8)


def silu(a):
    return a / (1 + np.exp(-a))


def gelu(a):
    return 0.5 * a * (1 + np.tanh(np.sqrt(2 / np.pi) * (a + 0.044715 * a ** 3)))
