"""Paged 8-bit key/value cache on the MI355X kernels: e4m3 blocks of 32 tokens with a power-of-two scale per block and
head, half the memory of the bf16 slot pools (host side of ``t2w_kv8_*``, ``include/t2w.h``; no counterpart in the reference,
whose pools are 16-bit, ``engine/runtime/dit_fast.py:59-64``).

A step over many requests is three calls on the caller's stream, none of which waits for the GPU or needs the lengths on the
host, so that one captured graph serves steps of any lengths::

    pages = KV8Pages.empty(n_blocks, kv_heads, head_dim)
    plan = KV8Plan(rows, n_tok)                                       # buffers, made once
    plan.build(kv_len, new_len, table, free_ids, free_head)           # block tables and slot maps
    append(pages, k, v, table, plan.row_start, plan.kv_total, max_new=longest)
    out = attention(q, pages, table, plan.row_start, plan.kv_total, scale=head_dim ** -0.5, chunk=1, max_new=longest, max_kv=bound)

``longest`` and ``bound`` are what the host knows of the rows' new and total tokens, 0 for nothing: they pick the kernel and its
split (a step of single tokens whose ``max_new`` is not said runs on tiles made for more).
The next step's ``kv_len`` and ``free_head`` are ``plan.kv_total`` and ``plan.free_head``; a plan's outputs must not be its own
inputs, so a loop alternates two plans or copies them.  Lengths, tables and ids are int32 tensors on the GPU.  No gradients
flow through these calls.
"""

from __future__ import annotations

import ctypes as C

import torch

from . import _lib

BLOCK = 32       # tokens of a block
MAX_ROWS = 4096  # rows of a call
# A step's calls take 4 to 8 us on the GPU: the host's part is kept as short.  torch's current stream of a device as the raw
# handle, without the 2 us of making a Stream object for each call; the current device likewise.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_I32 = torch.int32
_DTYPES = {torch.bfloat16: 0, torch.float16: 1}


def _small(what: str, n: int) -> None:
    if n > 0x7FFFFFFF:  # the struct's ints would wrap
        raise ValueError(f"kv8: {what} beyond 2^31 - 1")


class KV8Pages:
    """The cache's memory: ``k`` uint8 [n_blocks, kv_heads, head_dim / 16, 32, 16] (chunk of 16 channels, token, channel),
    ``v`` uint8 [n_blocks, kv_heads, 4, head_dim / 2, 2, 8] (8-token group, channel pair, channel, token), both e4m3 codes, and
    ``k_exp``, ``v_exp`` uint8 [n_blocks, kv_heads], the scales' exponents + 127.  The tensors stay the caller's."""

    __slots__ = ("k", "v", "k_exp", "v_exp", "n_blocks", "kv_heads", "head_dim", "device", "struct")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_exp: torch.Tensor, v_exp: torch.Tensor):
        if k.dim() != 5 or k.shape[3:] != (BLOCK, 16) or v.dim() != 6 or v.shape[2] != 4 or v.shape[4:] != (2, 8):
            raise ValueError("kv8 pages: k is [n_blocks, kv_heads, head_dim / 16, 32, 16], v [n_blocks, kv_heads, 4, head_dim / 2, 2, 8]")
        nb, g, c = k.shape[:3]
        d = 16 * c
        if v.shape[:2] != (nb, g) or v.shape[3] != d // 2 or k_exp.shape != (nb, g) or v_exp.shape != (nb, g):
            raise ValueError("kv8 pages: k, v, k_exp and v_exp differ in blocks, heads or channels")
        dev = k.device
        for t in (k, v, k_exp, v_exp):
            if t.dtype != torch.uint8 or not t.is_contiguous() or t.device != dev:
                raise ValueError("kv8 pages: contiguous uint8 tensors on one device")
        _small("n_blocks or kv_heads", max(nb, g))
        self.k, self.v, self.k_exp, self.v_exp = k, v, k_exp, v_exp
        self.n_blocks, self.kv_heads, self.head_dim, self.device = nb, g, d, dev
        self.struct = _lib.KV8Pages(k.data_ptr(), v.data_ptr(), k_exp.data_ptr(), v_exp.data_ptr(), nb, g, d)

    @classmethod
    def empty(cls, n_blocks: int, kv_heads: int, head_dim: int, device="cuda") -> "KV8Pages":
        """Pages of ``n_blocks`` blocks, zeroed."""
        if head_dim not in (64, 128):
            raise ValueError("kv8 pages: head_dim must be 64 or 128")
        z = lambda *s: torch.zeros(s, dtype=torch.uint8, device=device)  # noqa: E731
        return cls(z(n_blocks, kv_heads, head_dim // 16, BLOCK, 16), z(n_blocks, kv_heads, 4, head_dim // 2, 2, 8),
                   z(n_blocks, kv_heads), z(n_blocks, kv_heads))

    def values(self, ids=None) -> tuple[torch.Tensor, torch.Tensor]:
        """What blocks ``ids`` (all by default) hold: keys and values, fp32 [n, kv_heads, 32, head_dim]."""
        pick = (lambda t: t) if ids is None else (lambda t: t[ids])  # noqa: E731
        code = lambda t: pick(t).view(torch.float8_e4m3fn).float()  # noqa: E731

        def scaled(x, e):  # in two steps, each a normal power of two
            e = pick(e).float()[:, :, None, None]
            e = torch.where(e == 255, torch.nan, e - 127)  # E8M0's NaN
            half = torch.floor(e / 2)
            return x * torch.exp2(half) * torch.exp2(e - half)

        k = code(self.k).transpose(2, 3).flatten(3)
        v = code(self.v).permute(0, 1, 2, 5, 3, 4).flatten(4).flatten(2, 3)
        return scaled(k, self.k_exp), scaled(v, self.v_exp)


def _ints(what: str, t: torch.Tensor, n: int, dev) -> int:
    """Device pointer of a contiguous int32 vector of ``n`` entries."""
    if t.dtype is not _I32 or t.dim() != 1 or t.numel() != n or t.device != dev or not t.is_contiguous():
        raise ValueError(f"kv8: {what} must be a contiguous int32 vector of {n} on {dev}")
    return t.data_ptr()


def _table(t: torch.Tensor, rows: int, dev) -> tuple[int, int, int]:
    if t.dtype is not _I32 or t.dim() != 2 or t.device != dev:
        raise ValueError(f"kv8: the table must be int32 [{rows}, width] on {dev}")
    n, width = t.shape
    ld, one = t.stride()
    if n != rows or width < 1 or (one != 1 and width > 1):
        raise ValueError(f"kv8: the table must have {rows} rows, each contiguous")
    ld = ld if rows > 1 else width
    _small("the table's width or row stride", max(width, ld))
    return t.data_ptr(), width, ld


def _tokens(what: str, t: torch.Tensor, n, d: int, dev) -> int:
    """Elements between the token rows of [n_tok, heads, head_dim] (a token's heads lie side by side)."""
    if t.dim() != 3 or t.device != dev or t.dtype not in _DTYPES:
        raise ValueError(f"kv8: {what} must be bfloat16 or float16 [n_tok, heads, {d}] on {dev}")
    rows, heads, width = t.shape
    ld, head, one = t.stride()
    if width != d or one != 1 or (head != d and heads > 1):
        raise ValueError(f"kv8: {what} must be [n_tok, heads, {d}], a token's heads side by side")
    if n is not None and rows != n:
        raise ValueError(f"kv8: {what} must have {n} tokens")
    return ld if rows > 1 else heads * d


def _call(fn, args, dev, what: str) -> None:
    """One library call on torch's current stream of ``dev``."""
    if dev.type != "cuda":
        raise ValueError(f"kv8 {what}: the tensors must be on the GPU")
    if dev.index == _current_device():
        _lib.check(fn(C.byref(args), _raw_stream(dev.index)), what)
    else:
        with torch.cuda.device(dev):
            _lib.check(fn(C.byref(args), _raw_stream(dev.index)), what)


PLAN_ERRORS = {1: "a length is negative", 2: "more tokens than the plan has room for", 4: "a row outgrows its block table", 8: "too few free blocks"}


class KV8Plan:
    """Tables of a call over ``n_rows`` requests with room for ``n_tok`` new tokens, built on the GPU by ``build``:
    ``kv_total`` [n_rows], ``row_start`` [n_rows + 1], ``tok_row`` / ``tok_pos`` / ``slots`` [n_tok] (a token's row, position in
    its row, and block * 32 + place; -1 behind the last token), ``free_head`` [1], ``status`` [1].  The device-built counterpart of
    ``dit.plan_call``; buffers are reused by every ``build``."""

    def __init__(self, n_rows: int, n_tok: int, device="cuda"):
        if not 0 <= n_rows <= MAX_ROWS or n_tok < 0:
            raise ValueError(f"kv8 plan: 0 to {MAX_ROWS} rows, n_tok not negative")
        _small("n_tok", n_tok)
        self.n_rows, self.n_tok = int(n_rows), int(n_tok)
        sizes = (n_rows, n_rows + 1, n_tok, n_tok, n_tok, 1, 1)
        first = [0]
        for s in sizes:  # each at a 16-byte boundary
            first.append(first[-1] + (s + 3) // 4 * 4)
        buf = torch.empty(first[-1], dtype=torch.int32, device=device)
        self.device = buf.device
        views = [buf[a:a + s] for a, s in zip(first, sizes)]
        self.kv_total, self.row_start, self.tok_row, self.tok_pos, self.slots, self.free_head, self.status = views
        self._out = [buf.data_ptr() + 4 * a for a in first[:-1]]
        self._args = _lib.KV8PlanArgs(n_rows=self.n_rows, n_tok=self.n_tok)
        for (name, _), p in zip(_lib.KV8PlanArgs._fields_[-7:], self._out):
            setattr(self._args, name, p)

    def build(self, kv_len: torch.Tensor, new_len: torch.Tensor, table: torch.Tensor, free_ids: torch.Tensor, free_head: torch.Tensor) -> "KV8Plan":
        """Row r holds ``kv_len[r]`` tokens and gets ``new_len[r]``; the blocks it needs come from ``free_ids[free_head[0]:]`` in
        row order and go into ``table`` [n_rows, width] (only the new entries are written).  A call that cannot be served
        takes nothing and leaves rows without new tokens; ``check`` says why."""
        a, dev = self._args, self.device
        a.kv_len, a.new_len = _ints("kv_len", kv_len, self.n_rows, dev), _ints("new_len", new_len, self.n_rows, dev)
        a.table, a.width, a.ld_table = _table(table, self.n_rows, dev)
        _small("free_ids", free_ids.shape[0])
        a.n_free = free_ids.shape[0]
        a.free_ids = _ints("free_ids", free_ids, a.n_free, dev)
        a.free_head = _ints("free_head", free_head, 1, dev)
        _call(_lib.lib().t2w_kv8_plan, a, dev, "kv8_plan")
        return self

    def check(self) -> None:
        """Raises when the last ``build`` could not be served (waits for it)."""
        s = int(self.status.item())
        if s:
            raise RuntimeError("kv8 plan: " + ", ".join(text for bit, text in PLAN_ERRORS.items() if s & bit))


def append(pages: KV8Pages, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, row_start: torch.Tensor, kv_total: torch.Tensor,
           max_new: int = 0) -> None:
    """Quantizes the new tokens' keys and values, bf16 or fp16 [n_tok, kv_heads, head_dim] (rows may be strided: slices of
    a joint projection), into their rows' blocks.  ``max_new``: the longest row's new tokens if known (sizes the grid)."""
    dev, d, rows = pages.device, pages.head_dim, kv_total.shape[0]
    ldk, ldv = _tokens("k", k, None, d, dev), _tokens("v", v, k.shape[0], d, dev)
    _small("n_tok or max_new", max(k.shape[0], max_new))
    if k.dtype != v.dtype or k.shape[1] != pages.kv_heads or v.shape[1] != pages.kv_heads:
        raise ValueError(f"kv8 append: k and v of one type with {pages.kv_heads} heads")
    a = _lib.KV8AppendArgs(pages.struct, k.data_ptr(), v.data_ptr(), ldk, ldv, _DTYPES[k.dtype], k.shape[0], *_table(table, rows, dev),
                           _ints("row_start", row_start, rows + 1, dev), _ints("kv_total", kv_total, rows, dev), rows, max_new)
    _call(_lib.lib().t2w_kv8_append, a, dev, "kv8_append")


def attention(q: torch.Tensor, pages: KV8Pages, table: torch.Tensor, row_start: torch.Tensor, kv_total: torch.Tensor, *, scale: float,
              chunk: int = 0, max_new: int = 0, max_kv: int = 0, out: torch.Tensor | None = None,
              workspace: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q K^T) V of every new token ``q`` [n_tok, heads, head_dim] over its row's cache; ``heads`` is 1 to 16 times
    the pages' heads.  ``chunk``: 0 a token sees all of its row, c > 0 the row's earlier tokens and the new ones of its own and
    earlier chunks of c (1: causal).  ``max_new`` / ``max_kv``: bounds on the rows' new and total tokens, 0 unknown (a row
    of more than ``max_new`` may get NaN).  ``out`` may be ``q``; its rows behind the last token are left as they were, all of
    them after a plan that could not be served (an ``out`` made here is then uninitialised)."""
    dev, d, rows = pages.device, pages.head_dim, kv_total.shape[0]
    ldq = _tokens("q", q, None, d, dev)
    _small("n_tok, chunk, max_new or max_kv", max(q.shape[0], chunk, max_new, max_kv))
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        ldo = q.shape[1] * d
    else:
        ldo = _tokens("out", out, q.shape[0], d, dev)
        if out.dtype != q.dtype or out.shape[1] != q.shape[1]:
            raise ValueError("kv8 attention: out must have q's type and heads")
    L = _lib.lib()
    a = _lib.KV8AttentionArgs(pages.struct, q.data_ptr(), out.data_ptr(), ldq, ldo, _DTYPES[q.dtype], q.shape[0], q.shape[1],
                              *_table(table, rows, dev), _ints("row_start", row_start, rows + 1, dev),
                              _ints("kv_total", kv_total, rows, dev), rows, chunk, scale, max_new, max_kv)
    need = L.t2w_kv8_attention_workspace_bytes(C.byref(a))
    if workspace is None and need:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    if workspace is not None:
        if workspace.device != dev or not workspace.is_contiguous():
            raise ValueError("kv8 attention: a contiguous workspace on the pages' device")
        a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    _call(L.t2w_kv8_attention, a, dev, "kv8_attention")
    return out
