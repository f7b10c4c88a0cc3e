"""Rotary positions of several axes for queries and keys (host side of ``t2w_rope``, ``include/t2w.h``): text, images and video.  No
counterpart in the reference's Token2Wav path, whose DiT has no positional encoding; ``DiTConfig.rope_theta`` is the one-axis
option there.

A pair of channels turns by the token's position on the pair's axis times the pair's frequency.  Angles are integers, products of
the position with 64 bits of the frequency, and rounded to fp32 only for the sine and cosine: within 2^-26 turns at every int32
position.  Calls go on the caller's current stream, wait for nothing and can be captured; no gradients flow through
them::

    rope = Rope([theta ** (-2 * p / d) for p in range(d // 2)], axis=sections(16, 24, 24))   # once, with the model
    rope.apply(q, k, pos, q_out=q, k_out=k)                                                  # pos int32 [axes, n_tok]
"""

from __future__ import annotations

import math

import torch

from . import _lib

_I32 = torch.int32
_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
_PAIRS = {"halves": 0, "neighbours": 1}
# An angle's unit is 2^-64 turns, so one over the circle's number is needed far beyond a double: as an integer in units of 2^-_BITS
_BITS = 256
_PI_DIGITS = 314159265358979323846264338327950288419716939937510582097494459230781640628620899862  # pi 10^83
_PER_RADIAN = 10 ** 83 * 2 ** _BITS // (2 * _PI_DIGITS)


def _turns(f: float) -> int:
    """``f`` radians in turns of 2^-64, wrapped, as a signed 64-bit integer."""
    num, den = f.as_integer_ratio()  # den is a power of two
    shift = _BITS - 64 + den.bit_length() - 1
    t = (num * _PER_RADIAN + (1 << (shift - 1)) >> shift) & 0xFFFFFFFFFFFFFFFF
    return t - (1 << 64) if t >> 63 else t


def sections(*counts: int) -> list[int]:
    """Axis of every pair where the first ``counts[0]`` pairs count on axis 0, the next ``counts[1]`` on axis 1 and so on."""
    return [a for a, n in enumerate(counts) for _ in range(n)]


class Rope:
    """``inv_freq``: a frequency for every pair, radians a position (numbers; ``theta ** (-2 p / rot)`` in the plain form).  ``axis``: the
    axis each pair counts on (all on axis 0 by default).  ``pairs``: "halves" pairs channel p with p + rot / 2, "neighbours"
    2 p with 2 p + 1, where rot = 2 len(inv_freq) is a multiple of 16; a head's further channels keep their values.  ``scale``
    multiplies the turned channels."""

    __slots__ = ("rot", "n_axes", "pairs", "scale", "device", "_freq", "_axis")

    def __init__(self, inv_freq, axis=None, pairs: str = "halves", scale: float = 1.0, device="cuda"):
        inv = [float(f) for f in inv_freq]
        axis = [0] * len(inv) if axis is None else [int(a) for a in axis]
        if not inv or len(inv) % 8 or not all(abs(f) <= 2.0 ** 64 for f in inv):
            raise ValueError("rope: a multiple of 8 finite frequencies, at most 2^64")
        if len(axis) != len(inv) or min(axis) < 0 or max(axis) > 15:
            raise ValueError("rope: an axis (0 to 15) for every frequency")
        if pairs not in _PAIRS:
            raise ValueError("rope: pairs must be 'halves' or 'neighbours'")
        if not math.isfinite(scale):
            raise ValueError("rope: scale must be finite")
        self.rot, self.n_axes, self.pairs, self.scale = 2 * len(inv), max(axis) + 1, pairs, float(scale)
        n = len(inv)
        table = torch.tensor([_turns(f) for f in inv] + [int.from_bytes(bytes(axis[i:i + 8]), "little") for i in range(0, n, 8)], dtype=torch.int64).to(device)
        self._freq, self._axis = table[:n], table[n:].view(torch.uint8)  # the axes as bytes behind the frequencies
        self.device = self._freq.device

    def apply(self, q: torch.Tensor, k: torch.Tensor | None, pos: torch.Tensor, *, q_out: torch.Tensor | None = None,
              k_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
        """Turns ``q`` [n_tok, heads, head_dim] and ``k`` [n_tok, kv_heads, head_dim] (or None), bf16 or fp16, token rows strided by
        multiples of 8.  ``pos`` int32 [axes, n_tok] ([n_tok] for one axis; text, where all axes count alike,
        may be ``pos.expand(axes, n_tok)``), with at least the axes that the pairs count on.  The
        outputs, new tensors by default, may be ``q`` and ``k`` themselves."""
        dev, dtype = self.device, q.dtype
        code = _DTYPES.get(dtype)
        if code is None:
            raise ValueError("rope: q must be bfloat16 or float16")
        n, heads, d = q.shape if q.dim() == 3 else (0, 0, 0)
        ldq = _tokens("q", q, n, heads, d, dtype, dev)
        if pos.dim() == 1:
            pos = pos[None]
        shape = pos.shape
        if pos.dtype is not _I32 or len(shape) != 2 or shape[1] != n or pos.device != dev or (pos.stride(1) != 1 and n > 1):
            raise ValueError(f"rope: pos must be int32 [axes, {n}] on {dev}, each row contiguous")
        axes = self.n_axes
        if shape[0] < axes:
            raise ValueError(f"rope: pos must have the {axes} axes that the pairs count on")
        if q_out is None:
            q_out, ldo = torch.empty_like(q, memory_format=torch.contiguous_format), heads * d
        else:
            ldo = ldq if q_out is q else _tokens("q_out", q_out, n, heads, d, dtype, dev)
        if max(n, heads, d) > 0x7FFFFFFF:  # the struct's ints would wrap
            raise ValueError("rope: at most 2^24 tokens")
        kp = ko = None
        g = ldk = ldko = 0
        if k is not None:
            g = k.shape[1] if k.dim() == 3 else 0
            ldk = _tokens("k", k, n, g, d, dtype, dev)
            if k_out is None:
                k_out, ldko = torch.empty_like(k, memory_format=torch.contiguous_format), g * d
            else:
                ldko = ldk if k_out is k else _tokens("k_out", k_out, n, g, d, dtype, dev)
            kp, ko = k.data_ptr(), k_out.data_ptr()
        elif k_out is not None:
            raise ValueError("rope: k_out without k")
        a = _lib.RopeArgs(q.data_ptr(), kp, q_out.data_ptr(), ko, ldq, ldk, ldo, ldko, code, n, heads, g, d, self.rot, _PAIRS[self.pairs], self._freq.data_ptr(),
                          self._axis.data_ptr(), pos.data_ptr(), pos.stride(0) if axes > 1 else n, axes, self.scale)
        _lib.launch(_lib.lib().t2w_rope, a, dev, "rope")
        return q_out, k_out


def _tokens(what: str, t: torch.Tensor, n: int, heads: int, d: int, dtype, dev) -> int:
    """Elements between the token rows of [n_tok, heads, head_dim] (a token's heads lie side by side)."""
    if t.dtype is not dtype or t.dim() != 3 or t.device != dev:
        raise ValueError(f"rope: {what} must be {dtype} [n_tok, heads, head_dim] on {dev}")
    ld, head, one = t.stride()
    if t.shape != (n, heads, d) or one != 1 or (head != d and heads > 1):
        raise ValueError(f"rope: {what} must be [{n}, {heads}, {d}], a token's heads side by side")
    return ld if n > 1 else heads * d
