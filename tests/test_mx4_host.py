"""4-bit weights and rotary positions without a GPU: what their calls refuse, the oracle's code table and quantizer, the angles."""

import ctypes as C
import math
from fractions import Fraction

import numpy as np
import pytest
import torch

import t2w_amd  # noqa: F401
from oracle import mx4 as om
from oracle import rope as orp
from t2w_amd import _lib, mx4, rope

M = 1 << 20


def refused(fn, args, text):
    assert fn(C.byref(args), None) == 1
    assert text in _lib.lib().t2w_last_error().decode()


def weight(n=64, k=256, at=100, **kw):
    return _lib.MX4Weight(**({"codes": at * M, "scales": (at + 10) * M, "n": n, "k": k} | kw))


def linear_args(**kw):
    w = weight(**{x: kw.pop(x) for x in ("codes", "scales", "n", "k") if x in kw})
    return _lib.MX4LinearArgs(**({"x": 1 * M, "ldx": 256, "dtype": 0, "m": 4, "w": w, "bias": 2 * M, "residual": 3 * M, "ldr": 64, "y": 4 * M, "ldy": 64} | kw))


ROWS_BAD = [({"dtype": 2}, "dtype"), ({"m": -1}, "m must be"), ({"m": (1 << 20) + 1}, "m must be"), ({"x": None}, "null rows"), ({"y": None}, "null rows"),
            ({"x": M + 8}, "aligned"), ({"ldx": 260}, "aligned"), ({"y": 4 * M + 1}, "misaligned"), ({"ldx": 248}, "rows overlap"), ({"ldy": 63}, "rows overlap"),
            ({"y": M + 64}, "overlap x")]
LINEAR_BAD = ROWS_BAD + [({"n": 0}, "n must be"), ({"n": (1 << 24) + 1}, "n must be"), ({"k": 4}, "k must be"), ({"k": 252}, "k must be"), ({"k": (1 << 20) + 8}, "k must be"),
                         ({"codes": None}, "null weight"), ({"scales": None}, "null weight"), ({"codes": 100 * M + 8}, "aligned"), ({"scales": 110 * M + 2}, "aligned"),
                         ({"bias": 2 * M + 2}, "bias"), ({"residual": 3 * M + 1}, "misaligned"), ({"ldr": 60}, "rows overlap"),
                         ({"residual": 4 * M + 4}, "overlap the residual"), ({"residual": 4 * M, "ldr": 72}, "overlap the residual"),
                         ({"y": 2 * M + 128}, "weight or bias"), ({"y": 100 * M + 4}, "weight or bias")]


@pytest.mark.parametrize("kw,text", LINEAR_BAD, ids=str)
def test_linear_refuses(kw, text):
    refused(_lib.lib().t2w_mx4_linear, linear_args(**kw), text)


@pytest.mark.parametrize("kw,text", ROWS_BAD + [({"act": 2}, "act"), ({"up": weight(n=80, at=140)}, "sizes differ"), ({"up": weight(k=128, at=140)}, "sizes differ"),
                                                ({"gate": weight(codes=None)}, "null weight"), ({"y": 140 * M}, "overlap a weight")], ids=str)
def test_gated_refuses(kw, text):
    a = _lib.MX4GatedArgs(**({"x": M, "ldx": 256, "dtype": 0, "m": 4, "gate": weight(), "up": weight(at=140), "act": 0, "y": 4 * M, "ldy": 64} | kw))
    refused(_lib.lib().t2w_mx4_gated, a, text)


def ffn_args(**kw):
    return _lib.MX4FFNArgs(**({"x": M, "ldx": 256, "dtype": 1, "m": 4, "gate": weight(), "up": weight(at=140), "down": weight(n=256, k=64, at=180), "act": 1,
                               "residual": 2 * M, "ldr": 256, "y": 3 * M, "ldy": 256, "workspace": 5 * M, "workspace_bytes": 4 * 64 * 2} | kw))


@pytest.mark.parametrize("kw,text", [({"m": -1}, "m must be"), ({"act": -1}, "act"), ({"down": weight(n=256, k=72, at=180)}, "columns"), ({"up": weight(n=72, at=140)}, "sizes"),
                                     ({"down": weight(n=0, k=64)}, "n must be"), ({"ldy": 248}, "rows overlap"), ({"workspace": None}, "workspace too small"),
                                     ({"workspace_bytes": 511}, "workspace too small"), ({"workspace": 5 * M + 8}, "workspace must be"),
                                     ({"workspace": M}, "workspace overlaps"), ({"workspace": 3 * M}, "workspace overlaps"), ({"workspace": 2 * M + 16}, "workspace overlaps"),
                                     ({"workspace": 180 * M}, "workspace overlaps"), ({"y": 140 * M}, "overlap a weight"), ({"y": M}, "overlap x")], ids=str)
def test_ffn_refuses(kw, text):
    refused(_lib.lib().t2w_mx4_ffn, ffn_args(**kw), text)


def test_ffn_workspace():
    fn = _lib.lib().t2w_mx4_ffn_workspace_bytes
    assert fn(C.byref(ffn_args())) == 4 * 64 * 2
    assert fn(C.byref(ffn_args(gate=weight(n=100), up=weight(n=100)))) == 4 * 104 * 2  # rows at 16-byte boundaries
    assert fn(C.byref(ffn_args(m=-1))) == 0 and fn(C.byref(ffn_args(m=0))) == 0


def test_ffn_inner_values():
    """Rounded or wide; wide ones take two rows each, and the parts of a product of twice the rows."""
    L = _lib.lib()
    for kw, text in (({"inner": 2}, "inner must be"), ({"inner": -1}, "inner must be"), ({"inner": 1}, "workspace too small"), ({"inner": 1, "workspace_bytes": 1023}, "workspace too small"),
                     ({"inner": 1, "workspace_bytes": 1024, "workspace": 2 * M - 1008}, "workspace overlaps")):
        refused(L.t2w_mx4_ffn, ffn_args(**kw), text)
    assert L.t2w_mx4_ffn_workspace_bytes(C.byref(ffn_args(inner=1))) == 2 * 4 * 64 * 2
    down = weight(n=512, k=5000, at=300)
    f = ffn_args(m=40, gate=weight(5000, 256), up=weight(5000, 256, at=200), down=down, inner=1, ldy=512, ldr=512)
    parts = L.t2w_mx4_linear_workspace_bytes(C.byref(linear_args(m=80, n=512, k=5000, ldx=5000)))
    assert parts > 0 and L.t2w_mx4_ffn_workspace_bytes(C.byref(f)) == 2 * 40 * 5000 * 2 + parts
    with pytest.raises(ValueError, match="'wide' or 'rounded'"):
        mx4.ffn(torch.zeros(4, 256, dtype=torch.float16), fake(64, 256), fake(64, 256), fake(256, 64), inner="exact")


def test_workspaces():
    """None for few rows; beyond, bounded whatever the sizes; too small, misaligned or overlapping ones are refused."""
    L = _lib.lib()
    need = lambda **kw: L.t2w_mx4_linear_workspace_bytes(C.byref(linear_args(**kw)))  # noqa: E731
    assert need(m=1) == need(m=16) == need(m=0) == need(m=64, k=12) == 0  # (k=256: the rows fit the LDS)
    split = need(m=64, n=512, k=14336, ldx=14336, ldy=512, ldr=512)
    assert split > 0
    for m in (17, 64, 65, 200, 1000, 1 << 20):
        for n in (1, 100, 4096, 100000, 1 << 24):
            for k in (8, 1024, 14336, 1 << 20):
                assert need(m=m, n=n, k=k) <= 34 << 20
                g = _lib.MX4GatedArgs(x=M, ldx=k, dtype=0, m=m, gate=weight(n, k), up=weight(n, k), act=0, y=M, ldy=n)
                assert L.t2w_mx4_gated_workspace_bytes(C.byref(g)) <= 34 << 20
    big = {"m": 64, "n": 512, "k": 14336, "ldx": 14336, "ldy": 512, "ldr": 512}
    for kw, text in (({}, "too small"), ({"workspace": 50 * M, "workspace_bytes": split - 1}, "too small"), ({"workspace": 50 * M + 8, "workspace_bytes": split}, "aligned"),
                     ({"workspace": 4 * M, "workspace_bytes": split}, "workspace overlaps"), ({"workspace": M, "workspace_bytes": split}, "workspace overlaps"),
                     ({"workspace": 3 * M, "workspace_bytes": split}, "workspace overlaps"), ({"workspace": 100 * M, "workspace_bytes": split}, "workspace overlaps"),
                     ({"workspace": 2 * M - 16, "workspace_bytes": split}, "workspace overlaps")):
        refused(L.t2w_mx4_linear, linear_args(**(big | kw)), text)
    g = {"x": M, "ldx": 14336, "dtype": 0, "m": 64, "gate": weight(512, 14336), "up": weight(512, 14336, at=140), "act": 0, "y": 4 * M, "ldy": 512}
    need_g = L.t2w_mx4_gated_workspace_bytes(C.byref(_lib.MX4GatedArgs(**g)))
    for kw, text in (({}, "too small"), ({"workspace": 4 * M, "workspace_bytes": need_g}, "workspace overlaps"), ({"workspace": 140 * M, "workspace_bytes": need_g}, "workspace overlaps")):
        refused(L.t2w_mx4_gated, _lib.MX4GatedArgs(**(g | kw)), text)
    f = ffn_args(m=64, workspace=50 * M, workspace_bytes=64 * 64 * 2)
    assert L.t2w_mx4_ffn_workspace_bytes(C.byref(f)) >= 64 * 64 * 2


def test_forms():
    """What a product takes, and that only those in parts ask for memory."""
    L = _lib.lib()
    assert mx4.form(1, 6144, 4096) == mx4.form(16, 6144, 4096) == (0, 0, 1)
    assert mx4.form(4001, 6144, 4096) == (64, 256, 1) and mx4.form(2005, 14336, 4096, gated=True) == (64, 128, 1)
    assert mx4.form(70, 40, 256, ldx=1 << 24) == (0, 0, 1)  # rows too far apart for a tile
    for m in (1, 16, 17, 64, 200, 1000):
        for n in (31, 512, 6144):
            for k in (264, 4096, 14336):
                need = L.t2w_mx4_linear_workspace_bytes(C.byref(linear_args(m=m, n=n, k=k, ldx=k)))
                rows, channels, parts = mx4.form(m, n, k)
                assert need == (parts * (-(-m // rows) * rows) * (-(-n // channels) * channels) * 4 if parts > 1 else 0)
    for bad in ((0, 64, 64), ((1 << 21) + 1, 64, 64), (4, 0, 64), (4, 64, 60)):
        with pytest.raises(RuntimeError, match="mx4"):
            mx4.form(*bad)
    assert L.t2w_mx4_product_form(4, 64, 64, 64, 0, None) == 1


def test_weight_sizes():
    L = _lib.lib()
    assert (L.t2w_mx4_codes_bytes(1, 8), L.t2w_mx4_scales_bytes(1, 8)) == (1024, 256)
    assert (L.t2w_mx4_codes_bytes(17, 520), L.t2w_mx4_scales_bytes(17, 520)) == (2 * 5 * 1024, 2 * 2 * 256)
    assert L.t2w_mx4_codes_bytes(0, 8) == 0 and L.t2w_mx4_scales_bytes(4, 12) == 0


@pytest.mark.parametrize("kw,text", [({"n": 0}, "n must be"), ({"k": 12}, "k must be"), ({"codes": None}, "null"), ({"status": None}, "null"), ({"codes": M + 2}, "misaligned"),
                                     ({"w_codes": 3 * M + 4}, "misaligned")], ids=str)
def test_pack_refuses(kw, text):
    a = _lib.MX4PackArgs(**({"codes": M, "scales": 2 * M, "n": 4, "k": 64, "w_codes": 3 * M, "w_scales": 4 * M, "status": 5 * M} | kw))
    refused(_lib.lib().t2w_mx4_pack, a, text)


@pytest.mark.parametrize("kw,text", [({"dtype": 3}, "dtype"), ({"w": None}, "null"), ({"w": M + 2}, "misaligned"), ({"ldw": 56}, "overlap"), ({"k": 60}, "k must be")], ids=str)
def test_quantize_refuses(kw, text):
    a = _lib.MX4QuantizeArgs(**({"w": M, "ldw": 64, "dtype": 2, "n": 4, "k": 64, "w_codes": 3 * M, "w_scales": 4 * M, "status": 5 * M} | kw))
    refused(_lib.lib().t2w_mx4_quantize, a, text)


@pytest.mark.parametrize("kw", [{"w_codes": M}, {"w_codes": M + 112}, {"w_codes": M - 1008}, {"w_codes": 2 * M}, {"w_scales": M + 124}, {"w_scales": 2 * M + 4}, {"w_scales": 3 * M + 1020}, {"status": M + 4},
                                {"status": 2 * M + 4}, {"status": 3 * M + 512}, {"status": 4 * M + 252}], ids=str)
def test_layout_in_its_own_inputs_is_refused(kw):
    """Threads read codes and scales in another order than they write: laid out over its inputs a matrix would be any mixture."""
    base = {"codes": M, "scales": 2 * M, "n": 4, "k": 64, "w_codes": 3 * M, "w_scales": 4 * M, "status": 5 * M}
    refused(_lib.lib().t2w_mx4_pack, _lib.MX4PackArgs(**(base | kw)), "overlap")
    quant = {"w": M, "ldw": 96, "dtype": 2, "n": 4, "k": 64, "w_codes": 3 * M, "w_scales": 4 * M, "status": 5 * M}
    if not any(2 * M <= v < 2 * M + 64 for v in kw.values()):
        refused(_lib.lib().t2w_mx4_quantize, _lib.MX4QuantizeArgs(**(quant | kw)), "overlap")
    if "w_codes" in kw:
        refused(_lib.lib().t2w_mx4_quantize, _lib.MX4QuantizeArgs(**(quant | {"w": kw["w_codes"] + 512, "w_codes": kw["w_codes"]})), "overlap")


def test_calls_without_rows_do_nothing():
    assert _lib.lib().t2w_mx4_linear(C.byref(linear_args(m=0, x=None, y=None, residual=None, bias=None)), None) == 0
    assert _lib.lib().t2w_mx4_ffn(C.byref(ffn_args(m=0, workspace=None, workspace_bytes=0)), None) == 0


def test_rows_between_rows_do_not_overlap():
    """y in the gaps of x's rows, the residual in y's place, one row between many: refused for what is behind it (a weight without memory)."""
    for kw in ({"x": M, "ldx": 320, "y": M + 512, "ldy": 320}, {"residual": 4 * M, "ldr": 64}, {"m": 1, "x": M, "y": M + 512, "ldx": 8, "ldy": 1, "ldr": 0}):
        refused(_lib.lib().t2w_mx4_linear, linear_args(bias=2 * M + 2, **kw), "bias")
    for kw in ({"x": M, "ldx": 320, "y": M + 510, "ldy": 320}, {"x": M, "ldx": 320, "y": M + 514, "ldy": 320}, {"x": M, "ldx": 320, "y": M + 512, "ldy": 328}):
        refused(_lib.lib().t2w_mx4_linear, linear_args(bias=2 * M + 2, **kw), "overlap x")


# --- the Python calls ---

def test_weight_object_refuses():
    c, s = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    for a, b, text in ((c.int(), s, "uint8"), (c[0], s, "codes uint8"), (c, s[:, :1], r"scales must be \[4, 2\]"), (c[:, :2], s[:, :1], "multiple of 8"), (c[:0], s[:0], "n must be"),
                       (c, s, "on the GPU")):
        with pytest.raises(ValueError, match=text):
            mx4.MX4Weight(a, b)
    for w, text in ((torch.zeros(4, 64, dtype=torch.float64), "float32"), (torch.zeros(64), "float32"), (torch.zeros(4, 60), "multiple of 8"), (torch.zeros(4, 64), "on the GPU")):
        with pytest.raises(ValueError, match=text):
            mx4.MX4Weight.quantize(w)


def fake(n, k):
    """A weight's handle without memory, on the CPU: enough for the checks in front of a call."""
    w = mx4.MX4Weight.__new__(mx4.MX4Weight)
    w.n, w.k, w.device, w.struct = n, k, torch.device("cpu"), weight(n, k)
    return w


def test_linear_object_refuses():
    w, x = fake(64, 256), torch.zeros(4, 256, dtype=torch.bfloat16)
    for kw, text in (({"x": x.float()}, "bfloat16 or float16"), ({"x": x[:, :248]}, r"\[rows, 256\]"), ({"x": x.T.contiguous().T}, "each row"), ({"x": x[0]}, "x must be"),
                     ({"bias": torch.zeros(64).half()}, "bias"), ({"bias": torch.zeros(63)}, "bias"), ({"bias": torch.zeros(128)[::2]}, "bias"),
                     ({"residual": torch.zeros(4, 64)}, "residual"), ({"residual": torch.zeros(3, 64).bfloat16()}, r"residual must be \[4, 64\]"),
                     ({"out": torch.zeros(4, 64).half()}, "out must be"), ({"out": torch.zeros(64, 4).bfloat16().T}, "each row"), ({}, "on the GPU")):
        with pytest.raises(ValueError, match=text):
            mx4.linear(**({"x": x, "w": w} | kw))


def test_ffn_object_refuses():
    x = torch.zeros(4, 256, dtype=torch.float16)
    for kw, text in (({"act": "relu"}, "act"), ({"x": x.double()}, "bfloat16"), ({"residual": x.bfloat16()}, "residual"), ({"out": x[:2]}, "out must be"),
                     ({"workspace": torch.zeros(4, 64)[:, ::2]}, "workspace"), ({}, "on the GPU")):
        with pytest.raises(ValueError, match=text):
            mx4.ffn(**({"x": x, "gate": fake(64, 256), "up": fake(64, 256), "down": fake(256, 64)} | kw))
    with pytest.raises(ValueError, match="act"):
        mx4.gated(x, fake(64, 256), fake(64, 256), act="tanh")


# --- the oracle ---

def test_code_table():
    """All 16 codes against the format's bits: sign, two exponent bits of bias 1, one mantissa bit."""
    got = om.values(np.arange(0, 256, 17, dtype=np.uint8)[:, None], np.full((16, 1), 127, np.uint8))
    for c in range(16):
        e, m = c >> 1 & 3, c & 1
        want = (m / 2 if e == 0 else (1 + m / 2) * 2.0 ** (e - 1)) * (-1 if c & 8 else 1)
        assert (got[c] == want).all()


def test_quantizer():
    g = np.random.default_rng(0)
    w = g.standard_normal((40, 96)) * np.exp2(g.integers(-30, 12, (40, 3))).repeat(32, 1)
    c, s = om.quantize(w)
    e = s.astype(int) - 127
    top = np.abs(w.reshape(40, 3, 32)).max(-1)
    assert (top <= 6 * 2.0 ** e).all() and ((top > 3 * 2.0 ** e) | (e == om.EMIN)).all()
    step = np.where(np.abs(w) >= 4 * 2.0 ** e.repeat(32, 1), 2, np.where(np.abs(w) >= 2 * 2.0 ** e.repeat(32, 1), 1, 0.5)) * 2.0 ** e.repeat(32, 1)
    assert (np.abs(om.values(c, s) - w) <= step / 2).all()
    again = om.quantize(om.values(c, s))
    assert np.array_equal(om.values(*again), om.values(c, s))
    ties = np.array([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0]])
    assert om.values(*om.quantize(ties)).tolist() == [[0, 1, 1, 2, 2, 4, 4, 6]]
    assert om.quantize(np.zeros((1, 8)))[1].tolist() == [[127]]


# --- rotary positions ---

def rope_args(**kw):
    return _lib.RopeArgs(**({"q": M, "k": 2 * M, "q_out": 3 * M, "k_out": 4 * M, "ldq": 512, "ldk": 256, "ldq_out": 512, "ldk_out": 256, "dtype": 0, "n_tok": 4, "q_heads": 8, "k_heads": 4,
                             "head_dim": 64, "rot": 64, "pairs": 0, "freq": 5 * M, "axis": 6 * M, "pos": 7 * M, "ld_pos": 4, "n_axes": 3, "scale": 1.0} | kw))


@pytest.mark.parametrize("kw,text", [({"dtype": 2}, "dtype"), ({"pairs": 2}, "pairs"), ({"head_dim": 8}, "head_dim"), ({"head_dim": 68}, "head_dim"), ({"rot": 72}, "rotated"), ({"rot": 24}, "rotated"), ({"rot": 0}, "rotated"),
                                     ({"n_tok": -1}, "2^24"), ({"n_tok": (1 << 24) + 1, "ld_pos": 1 << 25}, "2^24"), ({"q_heads": -1}, "heads"), ({"k_heads": 4097}, "heads"), ({"n_axes": 0}, "axes"), ({"n_axes": 17}, "axes"),
                                     ({"ld_pos": 3}, "axes"), ({"scale": math.nan}, "scale"), ({"freq": None}, "null table"), ({"pos": None}, "null table"), ({"q": None}, "null heads"), ({"k_out": None}, "null heads"),
                                     ({"q": M + 8}, "aligned"), ({"ldk_out": 260}, "aligned"), ({"ldq": 504}, "rows overlap"), ({"q_out": M + 64}, "overlaps an input"), ({"q_out": M, "ldq_out": 520}, "overlaps an input"),
                                     ({"k_out": M}, "overlaps an input"), ({"k_out": 3 * M + 512}, "outputs overlap"), ({"k_out": 7 * M}, "positions")], ids=str)
def test_rope_refuses(kw, text):
    refused(_lib.lib().t2w_rope, rope_args(**kw), text)


def test_rope_without_work():
    assert _lib.lib().t2w_rope(C.byref(rope_args(n_tok=0, q=None)), None) == 0
    assert _lib.lib().t2w_rope(C.byref(rope_args(q_heads=0, k_heads=0, q=None, k=None)), None) == 0


def test_rope_rows_of_positions():
    """One row for all axes is taken (refused here for what is behind it), rows that overlap in part or run backwards are not."""
    refused(_lib.lib().t2w_rope, rope_args(ld_pos=0, freq=None), "null table")
    refused(_lib.lib().t2w_rope, rope_args(ld_pos=0, k_out=7 * M), "positions")
    for ld in (1, 3, -4):
        refused(_lib.lib().t2w_rope, rope_args(ld_pos=ld), "axes")


def test_rope_slices_of_one_projection():
    """In place on the query and key columns of one buffer: not refused for overlapping (but for the missing positions here)."""
    both = {"q": M, "k": M + 1024, "q_out": M, "k_out": M + 1024, "ldq": 1024, "ldk": 1024, "ldq_out": 1024, "ldk_out": 1024}
    refused(_lib.lib().t2w_rope, rope_args(pos=None, **both), "null table")
    refused(_lib.lib().t2w_rope, rope_args(**(both | {"k_out": M + 1008})), "overlap")
    refused(_lib.lib().t2w_rope, rope_args(**(both | {"k_out": M + 1040})), "overlaps an input")


def _arctan_inverse(x):
    """arctan(1 / x) in units of 10^-100, from its series."""
    total = term = 10 ** 100 // x
    n, sign = 3, -1
    while term:
        term //= x * x
        total += sign * (term // n)
        n, sign = n + 2, -sign
    return total


def test_rope_object():
    inv = [10000.0 ** (-2 * p / 64) for p in range(32)]
    r = rope.Rope(inv, device="cpu")
    for p in (0, 7, 31):  # the table's turns against the angle itself
        assert abs(int(r._freq[p]) / 2.0 ** 64 % 1 - inv[p] / (2 * math.pi) % 1) < 2 ** -52
    pi = 4 * (4 * _arctan_inverse(5) - _arctan_inverse(239))  # Machin's formula in units of 10^-100
    for f in (1.0, -0.5, 0.0, 1e-300, 5e-324, 1e-9, 12345.678, 2.0 ** 64):
        want = round(Fraction(f) * 10 ** 100 / (2 * pi) * 2 ** 64) % 2 ** 64
        assert rope._turns(f) % 2 ** 64 == want
    assert rope.sections(2, 0, 3) == [0, 0, 2, 2, 2]
    for kw, text in (({"inv_freq": inv[:7]}, "multiple of 8"), ({"inv_freq": []}, "multiple of 8"), ({"inv_freq": inv[:7] + [math.inf]}, "finite"), ({"inv_freq": inv[:7] + [math.nan]}, "finite"), ({"inv_freq": inv[:7] + [1e20]}, "2.64"), ({"inv_freq": inv, "axis": [0] * 31}, "axis"),
                     ({"inv_freq": inv, "axis": [0] * 31 + [16]}, "axis"), ({"inv_freq": inv, "axis": [-1] * 32}, "axis"), ({"inv_freq": inv, "pairs": "odd"}, "pairs"), ({"inv_freq": inv, "scale": math.nan}, "scale")):
        with pytest.raises(ValueError, match=text):
            rope.Rope(**({"device": "cpu"} | kw))
    r = rope.Rope(inv, axis=rope.sections(8, 12, 12), device="cpu")
    q, pos = torch.zeros(4, 8, 64, dtype=torch.float16), torch.zeros(3, 4, dtype=torch.int32)
    for kw, text in (({"q": q.float()}, "bfloat16"), ({"q": q[0]}, "q must be"), ({"q": q.transpose(0, 1).contiguous().transpose(0, 1)}, "side by side"), ({"k": q.bfloat16()}, "k must be"), ({"k": q[:3]}, "k must be"),
                     ({"pos": pos.long()}, "int32"), ({"pos": pos[:2]}, "3 axes"), ({"pos": pos[0]}, "3 axes"), ({"pos": pos[:, :3]}, "pos must be"), ({"pos": pos.T.contiguous().T}, "pos must be"),
                     ({"q_out": q[:, :4]}, "q_out"), ({"k": q, "k_out": q[:, :4]}, "k_out"), ({"k_out": q}, "without k"), ({}, "on the GPU")):
        with pytest.raises(ValueError, match=text):
            r.apply(**({"q": q, "k": None, "pos": pos} | kw))


def test_rope_oracle():
    """A turn by p then by -p is the identity; dot products depend on the distance of positions only."""
    g = np.random.default_rng(1)
    inv, axis = [100.0 ** (-p / 8) for p in range(8)], [0] * 3 + [1] * 5
    for pairs in ("halves", "neighbours"):
        x, pos = g.standard_normal((5, 2, 24)), g.integers(-1000, 1000, (2, 5))
        y = orp.rotate(x, pos, inv, axis, pairs)
        assert np.allclose(orp.rotate(y, -pos, inv, axis, pairs), x, atol=1e-12) and (y[..., 16:] == x[..., 16:]).all()
        a, b = x[:1], x[1:2]
        dot = [float((orp.rotate(a, p, inv, axis, pairs) * orp.rotate(b, p + 3, inv, axis, pairs)).sum()) for p in (pos[:, :1], pos[:, :1] + 17)]
        assert abs(dot[0] - dot[1]) < 1e-9
