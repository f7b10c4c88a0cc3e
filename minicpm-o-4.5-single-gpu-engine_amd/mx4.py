"""Linear layers and gated feed-forward blocks on 4-bit weights (host side of ``t2w_mx4_*``, ``include/t2w.h``): OCP MXFP4, e2m1
codes with a power-of-two scale for every 32 input columns, 4.25 bits a weight.  No counterpart in the reference, whose own reduced
weights are e4m3 (``engine/runtime/fp8.py:15-37``).

For callers that run the layers around the paged 8-bit cache (``t2w_amd.kv8``) on the same GPU::

    qkv_w = MX4Weight.quantize(w)                     # or MX4Weight(codes, scales) of a checkpoint; once, when a model is loaded
    qkv = linear(x, qkv_w, bias=b).view(n_tok, heads + 2 * kv_heads, head_dim)
    ...                                               # t2w_amd.rope, kv8.append, kv8.attention
    y = linear(o.flatten(1), o_w, residual=x)
    z = ffn(y, gate_w, up_w, down_w, residual=y)

Activations are bf16 or fp16; weights take their type without a rounding, sums are fp32, a block's inner values keep 16 bits of
precision over fp32's range (or x's type, where asked for).  Calls go on the caller's current
stream, wait for nothing and can be captured.  No gradients flow through them.
"""

from __future__ import annotations

import ctypes as C

import torch

from . import _lib

GROUP = 32         # columns that share a scale
EXPONENTS = -23, 13  # of the scales: every weight is exact in bf16 and fp16
_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
_WEIGHTS = _DTYPES | {torch.float32: 2}
_ACTS = {"silu": 0, "gelu": 1}
_INNER = {"rounded": 0, "wide": 1}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_F32 = torch.float32
IN_LDS = 4096      # columns of 16 rows that fit the LDS: such calls need no workspace


class MX4Weight:
    """A weight matrix [n, k] laid out for the kernels.  ``codes`` uint8 [n, k / 2] hold two e2m1 codes a byte, the even column in
    the lower nibble; ``scales`` uint8 [n, ceil(k / 32)] the exponents + 127 of every 32 columns, -23 to 13 (any on a group of
    zeros).  k is a multiple of 8.  Laying out waits for the GPU; the tensors are not kept."""

    __slots__ = ("n", "k", "device", "codes", "scales", "struct")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dim() != 2 or codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or scales.device != codes.device:
            raise ValueError("mx4 weight: codes uint8 [n, k / 2] and scales uint8 [n, ceil(k / 32)] on one device")
        n, k = codes.shape[0], 2 * codes.shape[1]
        if scales.shape != (n, -(-k // GROUP)):
            raise ValueError(f"mx4 weight: scales must be [{n}, {-(-k // GROUP)}] for {k} columns")
        codes, scales = codes.contiguous(), scales.contiguous()
        if codes.data_ptr() % 4:
            codes = codes.clone()
        status = self._empty(n, k, codes.device)
        a = _lib.MX4PackArgs(codes.data_ptr(), scales.data_ptr(), n, k, self.codes.data_ptr(), self.scales.data_ptr(), status.data_ptr())
        _lib.launch(_lib.lib().t2w_mx4_pack, a, self.device, "mx4_pack")
        if int(status.item()):
            raise ValueError(f"mx4 weight: a scale is out of 2^{EXPONENTS[0]} .. 2^{EXPONENTS[1]}")

    @classmethod
    def quantize(cls, w: torch.Tensor) -> "MX4Weight":
        """Rounds ``w`` [n, k] (bf16, fp16 or fp32; rows may be strided): a group's scale is the smallest power of two that keeps its
        largest magnitude within 6, codes are rounded to nearest, ties to even."""
        if w.dim() != 2 or w.dtype not in _WEIGHTS:
            raise ValueError("mx4 quantize: w must be bfloat16, float16 or float32 [n, k]")
        w = w.detach()
        if w.stride(1) != 1 and w.shape[1] > 1 or (w.shape[0] > 1 and w.stride(0) < w.shape[1]):
            w = w.contiguous()
        self = cls.__new__(cls)
        n, k = w.shape
        status = self._empty(n, k, w.device)
        a = _lib.MX4QuantizeArgs(w.data_ptr(), w.stride(0) if n > 1 else k, _WEIGHTS[w.dtype], n, k, self.codes.data_ptr(), self.scales.data_ptr(),
                                 status.data_ptr())
        _lib.launch(_lib.lib().t2w_mx4_quantize, a, self.device, "mx4_quantize")
        if int(status.item()):
            raise ValueError("mx4 quantize: a weight is not finite or beyond 49152")
        return self

    def _empty(self, n: int, k: int, device) -> torch.Tensor:
        L = _lib.lib()
        if not 0 < n <= 0x7FFFFFFF or not 0 < k <= 0x7FFFFFFF or not L.t2w_mx4_codes_bytes(n, k):
            raise ValueError("mx4 weight: n must be 1 to 2^24, k 8 to 2^20 and a multiple of 8")
        if device.type != "cuda":
            raise ValueError("mx4 weight: the tensors must be on the GPU")
        self.n, self.k, self.device = n, k, device
        self.codes = torch.empty(L.t2w_mx4_codes_bytes(n, k), dtype=torch.uint8, device=device)
        self.scales = torch.empty(L.t2w_mx4_scales_bytes(n, k), dtype=torch.uint8, device=device)
        self.struct = _lib.MX4Weight(self.codes.data_ptr(), self.scales.data_ptr(), n, k)
        return torch.zeros(1, dtype=torch.int32, device=device)

    def values(self) -> torch.Tensor:
        """What the codes and scales stand for, fp32 [n, k]."""
        blocks, steps, units = -(-self.n // 16), -(-self.k // 128), -(-self.k // 512)
        table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), dtype=_F32, device=self.device)
        c = self.codes.view(blocks, steps, 4, 16, 16)
        v = torch.stack([table[(c & 15).int()], table[(c >> 4).int()]], -1).flatten(-2)  # [block, step, group, channel, 32]
        e = self.scales.view(blocks, units, 4, 16, 4).permute(0, 1, 4, 2, 3).reshape(blocks, 4 * units, 4, 16)[:, :steps]
        v = v * torch.exp2(e.float() - 127)[..., None]
        return v.permute(0, 3, 1, 2, 4).reshape(16 * blocks, 128 * steps)[:self.n, :self.k].contiguous()


# A step's calls take 4 to 8 us on the GPU, about what the host needs for a call: the checks below look at each property once.

def _rows(what: str, t: torch.Tensor, m, width: int, dtype, dev) -> int:
    """Elements between the rows of [m, width]."""
    shape = t.shape
    if t.dtype is not dtype or len(shape) != 2 or t.device != dev:
        raise ValueError(f"mx4: {what} must be {dtype} [rows, {width}] on {dev}")
    ld, one = t.stride()
    if shape[1] != width or (m is not None and shape[0] != m) or (one != 1 and width > 1):
        raise ValueError(f"mx4: {what} must be [{'rows' if m is None else m}, {width}], each row contiguous")
    return ld if shape[0] > 1 else width


def _input(x: torch.Tensor, w: MX4Weight) -> tuple[int, int, int]:
    """x's pointer, row stride, type and rows: the first fields of a call's arguments."""
    dtype = x.dtype
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError("mx4: x must be bfloat16 or float16")
    ld, m = _rows("x", x, None, w.k, dtype, w.device), x.shape[0]
    if m > 0x7FFFFFFF:  # the struct's int would wrap
        raise ValueError("mx4: at most 2^20 rows")
    return x.data_ptr(), ld, code, m


def _output(x: torch.Tensor, m: int, n: int, out, dev) -> tuple[torch.Tensor, int]:
    if out is None:
        return x.new_empty((m, n)), n
    return out, _rows("out", out, m, n, x.dtype, dev)


def _residual(x: torch.Tensor, m: int, n: int, residual, dev) -> tuple:
    return (None, 0) if residual is None else (residual.data_ptr(), _rows("residual", residual, m, n, x.dtype, dev))


def _run(fn, workspace_bytes, a, dev, workspace, what: str) -> None:
    """A call with the caller's workspace or one of its own (``workspace_bytes`` None: the call needs none)."""
    if workspace is not None:
        if workspace.device != dev or not workspace.is_contiguous():
            raise ValueError("mx4: a contiguous workspace on the weights' device")
    elif workspace_bytes is not None:
        need = workspace_bytes(C.byref(a))
        if need:
            workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    if workspace is not None:
        a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    _lib.launch(fn, a, dev, what)


def linear(x: torch.Tensor, w: MX4Weight, *, bias: torch.Tensor | None = None, residual: torch.Tensor | None = None,
           out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """x w^T + bias + residual: ``x`` [rows, k] bf16 or fp16 (rows may be strided by multiples of 8, without overlap), ``bias`` fp32 [n],
    ``residual`` [rows, n] of x's type.  ``out`` may be ``residual``.  ``workspace``: memory for calls that make none
    (``t2w_mx4_linear_workspace_bytes``)."""
    dev, n = w.device, w.n
    rows = _input(x, w)
    m = rows[3]
    out, ldy = _output(x, m, n, out, dev)
    b = None
    if bias is not None:
        if bias.dtype is not _F32 or bias.shape != (n,) or bias.device != dev or not bias.is_contiguous():
            raise ValueError(f"mx4: bias must be a contiguous float32 vector of {n} on {dev}")
        b = bias.data_ptr()
    L = _lib.lib()
    a = _lib.MX4LinearArgs(*rows, w.struct, b, *_residual(x, m, n, residual, dev), out.data_ptr(), ldy)
    _run(L.t2w_mx4_linear, L.t2w_mx4_linear_workspace_bytes if m > 16 or w.k > IN_LDS else None, a, dev, workspace, "mx4_linear")
    return out


def form(rows: int, n: int, k: int, *, gated: bool = False, ldx: int | None = None) -> tuple[int, int, int]:
    """The kernel that a product of these sizes takes: (0, 0, 1) the one for few rows, else tiles of that many rows and output channels
    and the parts that k is split into.  A block's last product has 2 rows for each of x where its inner values are wide."""
    f = _lib.MX4Form()
    _lib.check(_lib.lib().t2w_mx4_product_form(rows, n, k, k if ldx is None else ldx, gated, C.byref(f)), "mx4_product_form")
    return f.tile_rows, f.tile_channels, f.parts


def _pair(gate: MX4Weight, up: MX4Weight, act: str) -> int:
    if act not in _ACTS:
        raise ValueError("mx4: act must be 'silu' or 'gelu'")
    if up.device != gate.device:
        raise ValueError("mx4: the weights must be on one device")
    return _ACTS[act]


def gated(x: torch.Tensor, gate: MX4Weight, up: MX4Weight, *, act: str = "silu", out: torch.Tensor | None = None,
          workspace: torch.Tensor | None = None) -> torch.Tensor:
    """act(x gate^T) * (x up^T) in one kernel; ``act`` is "silu" or "gelu" (the tanh form)."""
    k, rows, dev = _pair(gate, up, act), _input(x, gate), gate.device
    out, ldy = _output(x, rows[3], gate.n, out, dev)
    L = _lib.lib()
    a = _lib.MX4GatedArgs(*rows, gate.struct, up.struct, k, out.data_ptr(), ldy)
    _run(L.t2w_mx4_gated, L.t2w_mx4_gated_workspace_bytes if rows[3] > 16 or gate.k > IN_LDS else None, a, dev, workspace, "mx4_gated")
    return out


def ffn(x: torch.Tensor, gate: MX4Weight, up: MX4Weight, down: MX4Weight, *, act: str = "silu", residual: torch.Tensor | None = None,
        inner: str = "wide", out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """(act(x gate^T) * (x up^T)) down^T + residual.  ``inner`` "wide": the inner values are held to 2^-16 of their value over fp32's
    range; "rounded": to x's type (of fp16, beyond 65504 they are infinite), which halves the last product's operations.  ``out`` may be
    ``residual``."""
    if inner not in _INNER:
        raise ValueError("mx4: inner must be 'wide' or 'rounded'")
    k, rows, dev = _pair(gate, up, act), _input(x, gate), gate.device
    if down.device != dev:
        raise ValueError("mx4: the weights must be on one device")
    m, n = rows[3], down.n
    out, ldy = _output(x, m, n, out, dev)
    L = _lib.lib()
    a = _lib.MX4FFNArgs(*rows, gate.struct, up.struct, down.struct, k, _INNER[inner], *_residual(x, m, n, residual, dev), out.data_ptr(), ldy)
    _run(L.t2w_mx4_ffn, L.t2w_mx4_ffn_workspace_bytes, a, dev, workspace, "mx4_ffn")
    return out
