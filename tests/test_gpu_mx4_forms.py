"""Products with 4-bit weights in every form that a call can take, each named and asserted: the kernel of few rows, the four tiles, k whole
and in parts, blocks and their two products, workspaces of exactly the size asked for.

The operands are chosen so that fp32 sums are exact in any order: rows of -1, 0 and 1, codes with scales of neighbouring sizes, biases and
residuals in the same steps, and the absolute sum of a row's products below 2^24 steps (asserted).  The outputs have to equal the
exact sums rounded once: a column left out, taken twice or scaled wrongly shows, however many there are.
"""

import ctypes as C
import math

import pytest
import torch

import t2w_amd  # noqa: F401
from t2w_amd import _lib, mx4
from test_gpu_mx4 import BF, FP, U, gen, rand, rounding

pytestmark = pytest.mark.gpu
TABLE = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def columns(steps):
    """Columns of that many steps of 128, the last of them whole or not."""
    return 128 * steps - 8 * (steps % 3)


def decode(c, s):
    """Codes' and scales' values in float64."""
    table = torch.tensor(TABLE + tuple(-v for v in TABLE), dtype=torch.float64, device="cuda")
    n, half = c.shape
    v = table[torch.stack([c & 15, c >> 4], -1).view(n, 2 * half).int()]
    return v * torch.exp2(s.double() - 127).repeat_interleave(32, 1)[:, :2 * half]


def packed(c, s):
    return mx4.MX4Weight(c, s), decode(c, s)


def weight(n, k, seed, low=-1):
    """Any codes; scales 2^low to 2^(low + 2), so values in steps of 2^(low - 1)."""
    g = gen(seed)
    c = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    return packed(c, torch.randint(127 + low, 130 + low, (n, -(-k // 32)), generator=g, device="cuda", dtype=torch.uint8))


def signs(m, k, dt, seed):
    return torch.randint(-1, 2, (m, k), generator=gen(seed), device="cuda").to(dt)


def steps_of(n, count, step, seed):
    return torch.randint(-count, count + 1, (n,) if isinstance(n, int) else n, generator=gen(seed), device="cuda") * step


def exact_linear(m, n, k, dt, seed=0):
    """A product, with bias and residual, the residual in the outputs' place too, against the exact sums."""
    w, v = weight(n, k, seed + n + k)
    x, bias, res = signs(m, k, dt, seed), steps_of(n, 40, 0.25, 1).float(), steps_of((m, n), 60, 0.25, 2).to(dt)
    xd = x.double()
    assert ((xd.abs() @ v.abs().T).max().item() + 30) * 4 < 2 ** 24
    y = xd @ v.T
    assert torch.equal(mx4.linear(x, w), y.to(dt))
    y = (y + bias.double() + res.double()).to(dt)
    assert torch.equal(mx4.linear(x, w, bias=bias, residual=res), y)
    for pad, first in ((0, 0), (5, 3)):
        buf = torch.full((m + 2, n + pad), 9.0, dtype=dt, device="cuda")
        keep = buf.clone()
        out = buf[1:m + 1, first:first + n]
        out.copy_(res)
        mx4.linear(x, w, bias=bias, residual=out, out=out)
        keep[1:m + 1, first:first + n] = y
        assert torch.equal(buf, keep)
    assert y.abs().max() > 0


STEPS = list(range(1, 10)) + [14, 18]


@pytest.mark.parametrize("dt", [BF, FP], ids=str)
@pytest.mark.parametrize("tile,m,ns", [((0, 0), 1, (99, 2052)), ((0, 0), 16, (99, 100)), ((16, 128), 20, (99, 100)), ((32, 128), 257, (2001, 2004)), ((64, 128), 2100, (2050, 2052)),
                                       ((64, 256), 3000, (2050, 2052))], ids=str)
def test_whole_columns(dev, tile, m, ns, dt):
    """Every remainder of each tile's loop, k whole, with outputs in whole groups of four and not."""
    for steps in STEPS:
        n, k = ns[steps % 2], columns(steps)
        assert mx4.form(m, n, k) == (*tile, 1)
        exact_linear(m, n, k, dt, steps)
    for n in ns:  # the other remainder of n at one size of each parity
        exact_linear(m, n, columns(8), dt)
        exact_linear(m, n, columns(9), dt)


@pytest.mark.parametrize("dt", [BF, FP], ids=str)
@pytest.mark.parametrize("tile,sizes", [((16, 128), [(17, 31, 27, 6), (70, 32, 126, 25), (700, 31, 31, 5), (700, 31, 45, 5), (40, 1027, 113, 9)]),
                                        ((32, 128), [(130, 31, 116, 29), (700, 32, 41, 10), (700, 31, 67, 11), (1500, 31, 36, 5), (1500, 31, 46, 5), (1500, 31, 56, 5)]),
                                        ((64, 128), [(300, 1027, 65, 11), (3000, 32, 69, 10), (3000, 31, 85, 10), (3000, 258, 40, 3)]),
                                        ((64, 256), [(520, 2500, 43, 5), (200, 6000, 47, 5), (200, 6001, 51, 5)])], ids=str)
def test_columns_in_parts(dev, tile, sizes, dt):
    """Parts of 4 to 14 steps, of unequal lengths, in each tile."""
    for m, n, steps, parts in sizes:
        k = columns(steps)
        assert mx4.form(m, n, k) == (*tile, parts)
        exact_linear(m, n, k, dt, steps)


@pytest.mark.parametrize("dt", [BF, FP], ids=str)
@pytest.mark.parametrize("m,n,k", [(16, 40, 5464), (16, 2048, 5464), (6, 4090, 14336), (3, 130, 30000)])
def test_few_rows_too_long_for_the_lds(dev, m, n, k, dt):
    assert mx4.form(m, n, k) == (0, 0, 1)
    exact_linear(m, n, k, dt)


@pytest.mark.parametrize("m,tile", [(1, (16, 128)), (17, (32, 128))])
def test_most_columns(dev, m, tile):
    """2^20 columns, in the most parts there are; a result of zero, or without some columns, is far off."""
    n, k = 20, 1 << 20
    form = mx4.form(m, n, k)
    assert form == (*tile, 256)
    w, v = weight(n, k, 1)
    x = signs(m, k, BF, m)
    assert (x.double().abs() @ v.abs().T).max().item() * 4 < 2 ** 24
    y = x.double() @ v.T
    assert y.abs().median() > 500
    assert torch.equal(mx4.linear(x, w), y.to(BF))
    for at in (0, 127, 128, 4095, 4096, k // 2 - 1, k // 2, k - 128, k - 1):  # one column by itself, first and last of steps and parts
        x.zero_()
        x[:, at] = 1
        assert torch.equal(mx4.linear(x, w), v[:, at].to(BF).expand(m, n))


# --- gated blocks -----------------------------------------------------------------------------------------------------------------

def exact_gated(m, n, k, dt, act, seed=0):
    """Sums of both matrices exact; act's own calculation off by 8 u (1 + |t|) as in the gated block's other tests, the product and the
    output by a rounding each."""
    (g, vg), (u, vu) = weight(n, k, seed + n + k, -6), weight(n, k, seed + n + k + 1, -6)
    x = signs(m, k, dt, seed)
    a, b = x.double() @ vg.T, x.double() @ vu.T
    assert (x.double().abs() @ torch.maximum(vg.abs(), vu.abs()).T).max().item() * 128 < 2 ** 24
    # gelu's 1 + tanh(u) is 0 in 64 bits from u = -19 on; 2 / (1 + e^(-2 u)) is the same number without the cancellation
    f = a * torch.sigmoid(a if act == "silu" else 2 * (2 / math.pi) ** 0.5 * (a + 0.044715 * a ** 3))
    t = 3 * a.abs() + (a.abs() ** 3 if act == "gelu" else 0)
    h = f * b
    # 1 / (1 + 2^t) of more than 2^126 is subnormal in fp32, where the reciprocal instruction gives zero: |a| 2^-126 of act at most
    # (gelu: from a = -10 on, where it is below 10^-36), and a product in that range one step of 2^-149
    tol = 8 * U * (1 + t) * h.abs() + 2 * U * h.abs() + (a * b).abs() * 2.0 ** -126 + 2.0 ** -149
    got = mx4.gated(x, g, u, act=act)
    worst = ((got.double() - h).abs() / (tol + rounding(h.abs() + tol, dt))).flatten()
    assert worst.max() <= 1, (worst.max(), a.flatten()[worst.argmax()], b.flatten()[worst.argmax()], got.flatten()[worst.argmax()])


@pytest.mark.parametrize("dt", [BF, FP], ids=str)
@pytest.mark.parametrize("tile,m,ns", [((0, 0), 16, (99, 100)), ((16, 64), 20, (99, 100)), ((32, 64), 257, (1027, 1028)), ((64, 64), 520, (2050, 2052)), ((64, 128), 1500, (2050, 2052))], ids=str)
def test_gated_whole_columns(dev, tile, m, ns, dt):
    for steps in STEPS:
        n, k = ns[steps % 2], columns(steps)
        assert mx4.form(m, n, k, gated=True) == (*tile, 1)
        exact_gated(m, n, k, dt, "silu" if steps % 3 else "gelu", steps)


@pytest.mark.parametrize("dt", [BF, FP], ids=str)
@pytest.mark.parametrize("tile,sizes", [((16, 64), [(17, 31, 27, 6), (700, 32, 31, 5), (40, 514, 113, 9)]), ((32, 64), [(17, 258, 104, 26), (700, 31, 41, 10), (1500, 32, 46, 5)]),
                                        ((64, 64), [(300, 514, 65, 11), (3000, 31, 85, 10), (3000, 130, 40, 3)]), ((64, 128), [(130, 4099, 45, 5), (130, 4100, 51, 5)])], ids=str)
def test_gated_columns_in_parts(dev, tile, sizes, dt):
    for m, n, steps, parts in sizes:
        k = columns(steps)
        assert mx4.form(m, n, k, gated=True) == (*tile, parts)
        exact_gated(m, n, k, dt, "silu", steps)


# --- blocks -----------------------------------------------------------------------------------------------------------------------

def whole_numbers(m, inner, out, dt, seed=0):
    """A block of 64 input columns whose inner values are whole numbers of up to 11 bits, more than bf16 holds: gates of 46 to 82 (there
    1 + e^-a is 1 in fp32 and silu(a) is a) times up values of -12 to 12."""
    g = gen(seed + inner)

    def few(rows, first, top):
        """codes [rows, 64]: column 0 `first`, three of the upper 32 columns a whole number up to `top`"""
        c = torch.zeros(rows, 64, dtype=torch.uint8, device="cuda")
        c[:, 0] = first
        at = 32 + torch.rand(rows, 32, generator=g, device="cuda").argsort(1)[:, :3]
        code = torch.tensor([2, 4, 5, 6, 7], dtype=torch.uint8, device="cuda")[:top]
        c.scatter_(1, at, code[torch.randint(0, top, (rows, 3), generator=g, device="cuda")] + 8 * torch.randint(0, 2, (rows, 3), generator=g, device="cuda").to(torch.uint8))
        return c[:, 0::2] | (c[:, 1::2] << 4)

    scales = torch.tensor([131, 127], dtype=torch.uint8, device="cuda").expand(inner, 2).contiguous()
    gate, up = packed(few(inner, 6, 5), scales), packed(few(inner, 0, 4), scales)  # 4 * 2^4 = 64
    down = packed(torch.randint(0, 256, (out, inner // 2), generator=g, device="cuda", dtype=torch.uint8), torch.full((out, -(-inner // 32)), 122, dtype=torch.uint8, device="cuda"))
    x = signs(m, 64, dt, seed)
    x[:, 0] = 1
    res = steps_of((m, out), 60, 0.25, 2).to(dt)
    a, b = x.double() @ gate[1].T, x.double() @ up[1].T
    assert a.min() >= 46 and b.abs().max() <= 12
    h = a * b
    assert (h.abs() @ down[1].abs().T).max().item() * 64 + 64 * 15 < 2 ** 24  # steps of 2^-6
    y = h @ down[1].T
    return x, gate[0], up[0], down[0], res, y, (y + res.double()).to(dt)


def check_block(m, inner, out, dt, seed=0):
    x, g, u, d, res, y, want = whole_numbers(m, inner, out, dt, seed)
    assert torch.equal(mx4.ffn(x, g, u, d), y.to(dt))
    assert torch.equal(mx4.ffn(x, g, u, d, residual=res), want)
    buf = torch.full((m + 2, out + 5), 9.0, dtype=dt, device="cuda")
    keep = buf.clone()
    at = buf[1:m + 1, 3:3 + out]
    at.copy_(res)
    mx4.ffn(x, g, u, d, residual=at, out=at)
    keep[1:m + 1, 3:3 + out] = want
    assert torch.equal(buf, keep)
    assert torch.equal(mx4.ffn(x, g, u, d, residual=res, inner="rounded"), mx4.linear(mx4.gated(x, g, u), d, residual=res))


@pytest.mark.parametrize("dt", [BF, FP], ids=str)
@pytest.mark.parametrize("tile,m,outs", [((0, 0), 1, (99, 2052)), ((0, 0), 8, (99, 100)), ((16, 128), 10, (99, 100)), ((32, 128), 129, (2001, 2004)), ((64, 128), 1050, (2050, 2052)),
                                         ((64, 256), 1500, (2050, 2052))], ids=str)
def test_blocks_whole_columns(dev, tile, m, outs, dt):
    """Wide inner values through each form of the last product: two rows for each of x."""
    for steps in (1, 2, 3, 4, 5, 6, 7, 8, 9, 18):
        out, inner = outs[steps % 2], columns(steps)
        assert mx4.form(2 * m, out, inner) == (*tile, 1)
        check_block(m, inner, out, dt, steps)


@pytest.mark.parametrize("dt", [BF, FP], ids=str)
@pytest.mark.parametrize("tile,sizes", [((0, 0), [(8, 2048, 43, 1), (2, 130, 110, 1)]), ((16, 128), [(9, 31, 27, 6), (20, 512, 40, 10), (350, 32, 31, 5)]), ((32, 128), [(65, 31, 116, 29), (350, 32, 41, 10), (750, 31, 46, 5)]),
                                        ((64, 128), [(150, 1027, 65, 11), (1500, 31, 85, 10)]), ((64, 256), [(260, 2500, 43, 5), (100, 6001, 47, 5)])], ids=str)
def test_blocks_columns_in_parts(dev, tile, sizes, dt):
    for m, out, steps, parts in sizes:
        inner = columns(steps)
        assert mx4.form(2 * m, out, inner) == (*tile, parts)
        check_block(m, inner, out, dt)


@pytest.mark.parametrize("dt", [BF, FP], ids=str)
def test_inner_rows_beyond_32_bit_offsets(dev, dt):
    """Inner rows of 4.6 GB: every 100 rows of x repeat the first, and so do the outputs."""
    x, g, u, d, res, _, want = whole_numbers(100, 14344, 64, dt)
    assert 2 * 80000 * 14344 * 2 > 2 ** 32
    got = mx4.ffn(x.repeat(800, 1), g, u, d, residual=res.repeat(800, 1))
    assert torch.equal(got, want.repeat(800, 1))


# --- products in parts as programs call them ------------------------------------------------------------------------------------------

SPLIT = [(40, 512, 5000), (40, 14336, 264), (200, 264, 9224)]  # rows, hidden, inner: parts in the last product, in the gated one, in the last


def block(hidden, inner):
    return weight(inner, hidden, 1, -8)[0], weight(inner, hidden, 2, -8)[0], weight(hidden, inner, 3, -8)[0]


def in_parts(m, hidden, inner):
    return mx4.form(m, inner, hidden, gated=True)[2] > 1 or (mx4.form(m, hidden, inner)[2] > 1 and mx4.form(2 * m, hidden, inner)[2] > 1)


@pytest.mark.parametrize("inner_form", ["wide", "rounded"])
@pytest.mark.parametrize("m,hidden,inner", SPLIT)
def test_graphs_of_products_in_parts(dev, m, hidden, inner, inner_form):
    assert in_parts(m, hidden, inner)
    g, u, d = block(hidden, inner)
    x = rand((m, hidden), BF, 1)
    run = lambda: mx4.linear(mx4.ffn(x, g, u, d, residual=x, inner=inner_form), g)  # noqa: E731
    run()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append(run())
        graphs.append(graph)
    for seed in range(6):
        x.copy_(rand((m, hidden), BF, 10 + seed))
        graphs[seed % 2].replay()
        got = outs[seed % 2].clone()
        want = run()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and want.isfinite().all()


def test_two_streams_of_products_in_parts(dev):
    """Parts of several calls in flight at once, each in a workspace of its own."""
    calls = [(rand((m, hidden), BF, m), *block(hidden, inner)) for m, hidden, inner in SPLIT]
    want = [mx4.ffn(x, g, u, d, residual=x) for x, g, u, d in calls]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                for j in (range(3) if i == 0 else reversed(range(3))):
                    x, g, u, d = calls[j]
                    got.append((j, mx4.ffn(x, g, u, d, residual=x)))
    for s in streams:
        s.synchronize()
    assert all(torch.equal(y, want[j]) for j, y in got)


def need(fn, struct, x, w, y, **kw):
    """Bytes that the library asks for."""
    a = struct(x=x.data_ptr(), ldx=x.stride(0), dtype=0 if x.dtype is BF else 1, m=x.shape[0], y=y.data_ptr(), ldy=y.stride(0), **w, **kw)
    return getattr(_lib.lib(), fn)(C.byref(a))


def guarded(n):
    """A workspace of n bytes, what it lies in and where."""
    buf = torch.full((n + 8192,), 0x5A, dtype=torch.uint8, device="cuda")
    return buf, buf[4096:4096 + n]


@pytest.mark.parametrize("dt", [BF, FP], ids=str)
@pytest.mark.parametrize("m,hidden,inner", SPLIT + [(3, 520, 1000), (16, 2048, 5464), (600, 520, 1000)])
def test_workspaces_of_the_size_asked_for(dev, m, hidden, inner, dt):
    """Exactly as many bytes as the library asks for, and nothing around them is written."""
    g, u, d = block(hidden, inner)
    x, y = rand((m, hidden), dt, 1), torch.empty(m, hidden, dtype=dt, device="cuda")
    for form in ("wide", "rounded"):
        n = need("t2w_mx4_ffn_workspace_bytes", _lib.MX4FFNArgs, x, {"gate": g.struct, "up": u.struct, "down": d.struct}, y, inner=form == "wide")
        buf, ws = guarded(n)
        got = mx4.ffn(x, g, u, d, inner=form, workspace=ws)
        assert buf[:4096].eq(0x5A).all() and buf[4096 + n:].eq(0x5A).all()
        assert torch.equal(got, mx4.ffn(x, g, u, d, inner=form))
        with pytest.raises(RuntimeError, match="too small"):
            mx4.ffn(x, g, u, d, inner=form, workspace=ws[:n - 1])
    for x_, w in ((x, g), (rand((m, inner), dt, 2), d)):
        n = need("t2w_mx4_linear_workspace_bytes", _lib.MX4LinearArgs, x_, {"w": w.struct}, y)
        assert (n > 0) == (mx4.form(m, w.n, w.k)[2] > 1)
        if n:
            buf, ws = guarded(n)
            got = mx4.linear(x_, w, workspace=ws)
            assert buf[:4096].eq(0x5A).all() and buf[4096 + n:].eq(0x5A).all()
            assert torch.equal(got, mx4.linear(x_, w))
    n = need("t2w_mx4_gated_workspace_bytes", _lib.MX4GatedArgs, x, {"gate": g.struct, "up": u.struct}, torch.empty(m, inner, dtype=dt, device="cuda"))
    assert (n > 0) == (mx4.form(m, inner, hidden, gated=True)[2] > 1)
    if n:
        buf, ws = guarded(n)
        got = mx4.gated(x, g, u, workspace=ws)
        assert buf[:4096].eq(0x5A).all() and buf[4096 + n:].eq(0x5A).all()
        assert torch.equal(got, mx4.gated(x, g, u))
