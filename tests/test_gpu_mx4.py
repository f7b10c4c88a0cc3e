"""Products with 4-bit weights on the GPU against float64: layout, quantizer, linear layers, gated blocks.

Codes and scales have to be equal.  A weight is exact in bf16 and fp16 and a product of two such values exact in fp32, so a sum of
K products is off by at most K u of the products' absolute sum (u = 2^-24, an fp32 rounding, however the sum is ordered), each
further addition (bias, residual) by u of what it adds up, and the output by eps / 2 of its value, or half the type's smallest step
(fp16: 2^-25; bf16's lies below anything here).
The gated block: a relative error of the gate's and the up value's sums as above; act' is at most 1.13 (gelu; silu 1.1), its own
calculation (a product, exp2, reciprocal, a product; exp2's argument t rounded a few times) is off by 8 u (1 + |t|), |t| <= 3 |a| for silu and
3 |a| + |a|^3 for gelu; the product is one rounding.  The inner rounding adds eps / 2 of the inner value, or 2^-25 in fp16.
"""

import numpy as np
import pytest
import torch

import t2w_amd  # noqa: F401
from oracle import mx4 as om
from t2w_amd import mx4

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16
U = 2.0 ** -24


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def random_weight(n, k, seed, lo=-9, hi=-4):
    """Any codes, scales of many sizes: the handle and its values in float64."""
    g = gen(seed)
    c = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    s = torch.randint(127 + lo, 128 + hi, (n, -(-k // 32)), generator=g, device="cuda", dtype=torch.uint8)
    return mx4.MX4Weight(c, s), torch.from_numpy(om.values(c.cpu().numpy(), s.cpu().numpy())).cuda()


def rand(shape, dt, seed, size=1.0):
    return (torch.randn(shape, generator=gen(seed), device="cuda") * size).to(dt)


def rounding(y, dt):
    """Half a step of the output's type."""
    return torch.maximum(y.abs() * torch.finfo(dt).eps / 2, torch.tensor(2.0 ** -25 if dt is FP else 0.0, dtype=torch.float64, device="cuda"))


def product(x, v):
    """x v^T in float64 and what K fp32 additions can move it."""
    x = x.double()
    return x @ v.T, v.shape[1] * U * (x.abs() @ v.abs().T)


def check_linear(x, w, v, bias=None, residual=None, out=None):
    y, tol = product(x, v)
    for t in (bias, residual):
        if t is not None:
            y = y + t.double()
            tol = tol + U * (y.abs() + tol)
    got = mx4.linear(x, w, bias=bias, residual=residual, out=out)
    assert got.dtype == x.dtype and got.shape == y.shape
    tol = tol + rounding(y.abs() + tol, x.dtype)
    worst = ((got.double() - y).abs() / tol.clamp(min=1e-300)).max().item() if y.numel() else 0.0
    assert worst <= 1.0, worst
    return got


def act_of(a, act):
    return a * torch.sigmoid(a) if act == "silu" else torch.nn.functional.gelu(a, approximate="tanh")


def gated_reference(x, vg, vu, act):
    """Float64 inner values and their error before the rounding to x's type."""
    (a, ta), (b, tb) = product(x, vg), product(x, vu)
    f = act_of(a, act)
    t = 3 * a.abs() + (a.abs() ** 3 if act == "gelu" else 0)
    tf = 1.13 * ta + 8 * U * (1 + t) * f.abs()
    h = f * b
    return h, tf * (b.abs() + tb) + f.abs() * tb + U * h.abs()


# --- layout ----------------------------------------------------------------------------------------------------------------

SIZES = [(1, 8), (5, 40), (16, 128), (17, 136), (100, 520), (257, 1032), (64, 2048)]


@pytest.mark.parametrize("n,k", SIZES)
def test_layout_holds_the_values(dev, n, k):
    w, v = random_weight(n, k, n + k, -23, 13)
    assert torch.equal(w.values().double(), v)


def test_layout_refuses_scales(dev):
    c, s = torch.full((20, 64), 0x11, dtype=torch.uint8, device="cuda"), torch.full((20, 4), 127, dtype=torch.uint8, device="cuda")
    for byte, ok in ((104, True), (140, True), (103, False), (141, False), (0, False), (255, False)):
        t = s.clone()
        t[17, 3] = byte
        if ok:
            assert mx4.MX4Weight(c, t).values()[17, 96:].eq(0.5 * 2.0 ** (byte - 127)).all()
            continue
        with pytest.raises(ValueError, match="scale"):
            mx4.MX4Weight(c, t)
        z = c.clone()
        z[17, 48:] = 0x08  # zeros of both signs
        assert mx4.MX4Weight(z, t).values()[17, 96:].eq(0).all()


def test_layout_of_slices(dev):
    c = torch.randint(0, 256, (40, 70), dtype=torch.uint8, device="cuda")
    s = torch.full((40, 5), 120, dtype=torch.uint8, device="cuda")
    w = mx4.MX4Weight(c[3:30, 2:66], s[3:30, :4])
    assert torch.equal(w.values().double().cpu(), torch.from_numpy(om.values(c[3:30, 2:66].cpu().numpy(), s[3:30, :4].cpu().numpy())))
    flat = torch.randint(0, 256, (8 * 32 + 1,), dtype=torch.uint8, device="cuda")[1:].view(8, 32)  # contiguous, not at 4 bytes
    assert torch.equal(mx4.MX4Weight(flat, s[:8, :2]).values(), mx4.MX4Weight(flat.clone(), s[:8, :2]).values())


@pytest.mark.parametrize("dt", [BF, FP, torch.float32], ids=str)
@pytest.mark.parametrize("n,k", SIZES)
def test_quantize(dev, n, k, dt):
    g = gen(n * k)
    size = torch.exp2(torch.randint(-28, 3, (n, -(-k // 8)), generator=g, device="cuda").float()).repeat_interleave(8, 1)[:, :k]
    w = (torch.randn(n, k, generator=g, device="cuda") * size).to(dt)
    w[0, :8] = torch.tensor([0.25, -0.75, 1.25, -1.75, 2.5, -3.5, 5.0, 6.0]).to(dt)  # ties, where no larger value shares their group
    want = om.values(*om.quantize(w.double().cpu().numpy()))
    assert torch.equal(mx4.MX4Weight.quantize(w).values().double().cpu(), torch.from_numpy(want))


def test_quantize_limits(dev):
    w = torch.zeros(3, 64, device="cuda")
    w[1, 5], w[2, 40] = 49152.0, 2.0 ** -24
    assert torch.equal(mx4.MX4Weight.quantize(w).values(), w)
    strided = torch.randn(16, 300, device="cuda")[::2, 4:260]
    for t in (strided, strided.T):
        assert torch.equal(mx4.MX4Weight.quantize(t).values(), mx4.MX4Weight.quantize(t.contiguous()).values())
    for bad in (float("nan"), float("inf"), -float("inf"), 49200.0):
        w[0, 3] = bad
        with pytest.raises(ValueError, match="finite"):
            mx4.MX4Weight.quantize(w)


# --- linear -------------------------------------------------------------------------------------------------------------------

ROWS = [1, 2, 3, 15, 16, 17, 33, 64, 65, 127, 129, 200, 256, 257, 520]


@pytest.mark.parametrize("dt", [BF, FP], ids=str)
@pytest.mark.parametrize("m", ROWS)
def test_linear_rows(dev, m, dt):
    for n, k in ((257, 1032), (96, 520)):
        w, v = random_weight(n, k, m + n)
        check_linear(rand((m, k), dt, m), w, v, bias=torch.randn(n, device="cuda"), residual=rand((m, n), dt, m + 1))


@pytest.mark.parametrize("dt", [BF, FP], ids=str)
@pytest.mark.parametrize("m", [1, 17, 70, 300])
@pytest.mark.parametrize("n,k", SIZES + [(31, 8192), (600, 14336), (1040, 264)])
def test_linear_sizes(dev, n, k, m, dt):
    w, v = random_weight(n, k, n + k + m)
    check_linear(rand((m, k), dt, m), w, v)


@pytest.mark.parametrize("dt", [BF, FP], ids=str)
@pytest.mark.parametrize("m,n,k", [(16, 40, 5464), (16, 300, 4096), (16, 1027, 14336), (9, 100, 9224), (40, 130, 14336), (3000, 31, 14336), (100, 4100, 9000), (257, 2001, 1032), (257, 31, 14336), (2000, 515, 264), (2000, 1027, 5000),
                                   (600, 4100, 5000), (4100, 6000, 1032)])
def test_linear_forms(dev, m, n, k, dt):
    """Sizes at which each form is chosen: rows too long for the LDS, the four tiles, with k whole and in parts."""
    w, v = random_weight(n, k, n + k + m)
    check_linear(rand((m, k), dt, m), w, v, bias=torch.randn(n, device="cuda"), residual=rand((m, n), dt, m + 1))


@pytest.mark.parametrize("m,n", [(1, 96), (20, 96), (257, 2001), (3000, 96), (3000, 515)])
@pytest.mark.parametrize("steps", list(range(1, 19)) + [27, 30])
def test_every_number_of_steps(dev, m, n, steps):
    """Columns of 1 to 30 steps of 128: every remainder of the loops, in calls of one row and in those that each of the tiles takes."""
    k = 128 * steps - 8 * (steps % 3)
    w, v = random_weight(n, k, steps)
    x = rand((m, k), FP, m)
    y = check_linear(x, w, v)
    assert all(torch.equal(mx4.linear(x, w), y) for _ in range(3))


@pytest.mark.parametrize("m", [1, 17])
def test_most_columns(dev, m):
    w, v = random_weight(20, 1 << 20, 1)
    check_linear(rand((m, 1 << 20), BF, m), w, v)


@pytest.mark.parametrize("dt", [BF, FP], ids=str)
@pytest.mark.parametrize("m", [1, 16, 40, 150, 400])
def test_linear_strides(dev, m, dt):
    """Rows of wider buffers, outputs at odd strides and offsets, the residual in the outputs' place."""
    n, k = 130, 264
    w, v = random_weight(n, k, m)
    x = rand((m, k + 72), dt, m)[:, 16:16 + k]
    for pad, first in ((0, 0), (6, 2), (7, 3), (2, 1)):
        buf = rand((m + 2, n + pad), dt, 5)
        keep = buf.clone()
        out = buf[1:m + 1, first:first + n]
        check_linear(x, w, v, residual=rand((m, n + 3), dt, 9)[:, 1:n + 1], out=out)
        keep[1:m + 1, first:first + n] = out
        assert torch.equal(buf, keep)  # nothing beside the rows
        want = check_linear(x, w, v, residual=out.clone())
        assert torch.equal(mx4.linear(x, w, residual=out, out=out), want)


@pytest.mark.parametrize("dt", [BF, FP], ids=str)
@pytest.mark.parametrize("m", [2, 20, 100, 300])
def test_values_that_are_not_finite_stay_in_their_rows(dev, m, dt):
    n, k = 200, 392  # the last step of columns is partly beyond k
    w, v = random_weight(n, k, 3)
    x = rand((m, k), dt, 4)
    want = check_linear(x, w, v)
    wg, _ = random_weight(n, k, 6)
    inner = mx4.gated(x, w, wg)
    bad = x.clone()
    bad[1, 390], bad[0, 0] = float("nan"), float("inf")
    got, gi = mx4.linear(bad, w), mx4.gated(bad, w, wg)
    assert torch.equal(got[2:], want[2:]) and torch.equal(gi[2:], inner[2:])
    assert got[1].isnan().all() and gi[1].isnan().all()
    col = v[:, 0]
    assert torch.equal(got[0].double(), torch.where(col == 0, torch.nan, torch.sign(col) * torch.inf).nan_to_num(nan=7e9)) or \
        torch.equal(got[0].double().nan_to_num(nan=7e9), torch.where(col == 0, torch.nan, torch.sign(col) * torch.inf).nan_to_num(nan=7e9))


@pytest.mark.parametrize("dt", [BF, FP], ids=str)
@pytest.mark.parametrize("m", [1, 30, 130, 300])
def test_small_and_large_values(dev, m, dt):
    """Weights and rows at the ends of fp16's range, subnormal ones among them."""
    n, k = 48, 256
    for lo, hi, size in ((-23, -22, 1.0), (-23, -20, 2.0 ** 12), (11, 13, 2.0 ** -18), (-23, 13, 2.0 ** -12)):
        w, v = random_weight(n, k, m, lo, hi)
        x = rand((m, k), dt, m, size)
        y = (x.double() @ v.T).abs().max().item()
        if dt is FP and y > 60000:
            x = x * (2.0 ** -10)
        check_linear(x, w, v)


def test_linear_beyond_32_bit_offsets(dev):
    """Outputs, inputs and codes whose places pass 2^31 elements or 2^32 bytes."""
    n, k, m = (1 << 20) + 5, 64, 2100
    w, v = random_weight(n, k, 1)
    x = rand((m, k), BF, 2)
    y = mx4.linear(x, w)
    for a, b in ((0, 40), (1 << 19, (1 << 19) + 40), (n - 40, n)):
        ref, tol = product(x, v[a:b])
        assert ((y[:, a:b].double() - ref).abs() <= tol + rounding(ref.abs() + tol, BF)).all()
    del y, w, v
    n, k, m = 40, 256, 1100
    w, v = random_weight(n, k, 3)
    x = torch.zeros(m, 1 << 21, dtype=BF, device="cuda")[:, (1 << 21) - k:]
    x.copy_(rand((m, k), BF, 4))
    check_linear(x, w, v)
    del x
    n, k = (1 << 20) + 40, 8448
    c = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda")
    s = torch.full((n, k // 32), 120, dtype=torch.uint8, device="cuda")
    w = mx4.MX4Weight(c, s)
    tail = torch.from_numpy(om.values(c[-60:].cpu().numpy(), s[-60:].cpu().numpy())).cuda()
    for m in (1, 200):
        x = rand((m, k), BF, m)
        ref, tol = product(x, tail)
        assert ((mx4.linear(x, w)[:, -60:].double() - ref).abs() <= tol + rounding(ref.abs() + tol, BF)).all()


def test_rows_far_apart(dev):
    """Rows of x more than 2^24 elements apart, whose places in a tile would pass a 32-bit offset, and just below."""
    n, k, m = 40, 256, 70
    w, v = random_weight(n, k, 3)
    for ld in ((1 << 24) - 8, 1 << 24):
        x = torch.zeros(m, ld, dtype=BF, device="cuda")[:, ld - k:]
        x.copy_(rand((m, k), BF, 4))
        check_linear(x, w, v)
        check_linear(x[:9], w, v)


def test_no_rows(dev):
    w, _ = random_weight(48, 64, 1)
    x = torch.empty(0, 64, dtype=BF, device="cuda")
    assert mx4.linear(x, w).shape == (0, 48) and mx4.ffn(x, w, w, random_weight(64, 48, 2)[0]).shape == (0, 64)


# --- gated blocks ----------------------------------------------------------------------------------------------------------------

def check_gated(m, n, k, dt, act):
    (g, vg), (u, vu) = random_weight(n, k, m), random_weight(n, k, m + 1)
    x = rand((m, k), dt, m, 8 * k ** -0.5)  # gates and products within fp16's range at every k
    h, tol = gated_reference(x, vg, vu, act)
    got = mx4.gated(x, g, u, act=act)
    tol = tol + rounding(h.abs() + tol, dt)
    assert ((got.double() - h).abs() <= tol).all()


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dt", [BF, FP], ids=str)
@pytest.mark.parametrize("m", ROWS)
def test_gated(dev, m, dt, act):
    for n, k in ((264, 520), (77, 1032)):
        check_gated(m, n, k, dt, act)


@pytest.mark.parametrize("dt", [BF, FP], ids=str)
@pytest.mark.parametrize("m,n,k", [(16, 40, 5464), (16, 5000, 4096), (16, 700, 14336), (40, 130, 14336), (50, 4100, 264), (257, 130, 14336), (3000, 31, 14336), (3000, 130, 264), (3000, 1027, 264), (257, 4100, 5000)])
def test_gated_forms(dev, m, n, k, dt):
    check_gated(m, n, k, dt, "silu")


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dt", [BF, FP], ids=str)
@pytest.mark.parametrize("m,hidden,inner", [(1, 256, 704), (3, 512, 1368), (16, 128, 8), (50, 264, 1000), (130, 256, 520), (300, 640, 1048)])
def test_ffn(dev, m, hidden, inner, dt, act):
    (g, vg), (u, vu), (d, vd) = random_weight(inner, hidden, 1), random_weight(inner, hidden, 2), random_weight(hidden, inner, 3)
    x, res = rand((m, hidden), dt, m), rand((m, hidden), dt, m + 1)
    h, th = gated_reference(x, vg, vu, act)
    th = th + rounding(h.abs() + th, dt)
    y, tol = product(h, vd)
    tol = tol + th @ vd.abs().T * (1 + inner * U)
    y = y + res.double()
    tol = tol + U * (y.abs() + tol)
    tol = tol + rounding(y.abs() + tol, dt)
    got = mx4.ffn(x, g, u, d, act=act, residual=res)
    assert ((got.double() - y).abs() <= tol).all()
    own = res.clone()
    assert torch.equal(mx4.ffn(x, g, u, d, act=act, residual=own, out=own, workspace=torch.empty(2 * m * inner + (36 << 20), dtype=torch.uint8, device="cuda")), got)


def test_gate_far_from_zero(dev):
    """Gates of any size: act(-large) is zero and act(large) the gate, with no infinity times zero between."""
    w = mx4.MX4Weight.quantize(torch.eye(16, device="cuda"))
    big = torch.tensor([0.0, 1e-4, -1e-4, 30, -30, 100, -100, 1000, -1000, 3e4, -3e4, 1e6, -1e6, 1e18, -1e18, 5], device="cuda")
    x = torch.diag(big).to(BF)
    one = mx4.MX4Weight.quantize(torch.ones(16, 16, device="cuda"))
    for act in ("silu", "gelu"):
        got = mx4.gated(x, w, one, act=act)
        v = x.diag().double()
        # the gate is x's diagonal entry, the up value the row's only entry
        want = act_of(v, act) * v
        assert torch.allclose(got.diag().double(), want, rtol=2.0 ** -7, atol=1e-9), act
        assert got.isfinite().all()


# --- calls as programs make them -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("m", [1, 24, 140, 300])
def test_rows_do_not_depend_on_their_neighbours(dev, m):
    """A call twice gives the same bits, and a row alone in its call's place keeps them whatever the other rows hold."""
    w, _ = random_weight(300, 1032, 1)
    x = rand((m, 1032), BF, 2)
    y = mx4.linear(x, w)
    assert torch.equal(mx4.linear(x, w), y)
    other = rand((m, 1032), BF, 3)
    other[m // 2] = x[m // 2]
    assert torch.equal(mx4.linear(other, w)[m // 2], y[m // 2])


@pytest.mark.parametrize("m", [1, 40, 300])
def test_other_stream_and_graph(dev, m):
    (g, _), (u, _), (d, _) = random_weight(520, 256, 1), random_weight(520, 256, 2), random_weight(256, 520, 3)
    x = rand((m, 256), BF, 1)
    want = mx4.ffn(x, g, u, d, residual=x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mx4.ffn(x, g, u, d, residual=x)
    side.synchronize()
    assert torch.equal(got, want)
    graphs, outs = [], []
    for _ in range(2):  # two graphs of one pool run in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append(mx4.linear(mx4.ffn(x, g, u, d, residual=x), g))
        graphs.append(graph)
    for seed in range(4):
        x.copy_(rand((m, 256), BF, 10 + seed))
        graphs[seed % 2].replay()
        eager = mx4.linear(mx4.ffn(x, g, u, d, residual=x), g)
        torch.cuda.synchronize()
        assert torch.equal(outs[seed % 2], eager)


def test_two_streams_at_once(dev):
    """Calls of several forms in flight on two streams, each with workspaces of its own."""
    (g, _), (u, _), (d, _) = random_weight(1400, 520, 1), random_weight(1400, 520, 2), random_weight(520, 1400, 3)
    xs = [rand((m, 520), BF, m) for m in (1, 16, 70, 700)]
    want = [mx4.ffn(x, g, u, d, residual=x) for x in xs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = {}
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for turn in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                for j in (range(4) if i == 0 else reversed(range(4))):
                    got[i, j, turn] = mx4.ffn(xs[j], g, u, d, residual=xs[j])
    for s in streams:
        s.synchronize()
    assert all(torch.equal(y, want[j]) for (_, j, _), y in got.items())


def test_inputs_are_read_only(dev):
    """Weights, rows, bias and residual keep their bytes, and so does what lies around a workspace."""
    (g, _), (u, _), (d, _) = random_weight(1000, 520, 1), random_weight(1000, 520, 2), random_weight(520, 1000, 3)
    for m in (3, 50, 600):
        x, r = rand((m, 520), FP, m), rand((m, 520), FP, 1)
        ws = torch.full((2 * m * 1000 + (40 << 20),), 0x5A, dtype=torch.uint8, device="cuda")
        keep = [t.clone() for t in (x, r, g.codes, g.scales, u.codes, d.codes, d.scales)]
        need = 2 * m * 1000 + (34 << 20)
        mx4.ffn(x, g, u, d, residual=r, workspace=ws[:need])
        assert all(torch.equal(a, b) for a, b in zip((x, r, g.codes, g.scales, u.codes, d.codes, d.scales), keep))
        assert ws[need:].eq(0x5A).all()


@pytest.mark.parametrize("m,k", [(1, 392), (7, 8), (16, 136), (20, 8), (40, 392), (333, 1032), (3000, 200), (200, 5000)])
def test_nothing_of_an_earlier_call_is_left_behind(dev, m, k):
    """Rows and columns beyond a call's end read as zeros although the LDS of every CU holds NaN of the call before."""
    w, _ = random_weight(300, k, 1)
    big, _ = random_weight(4096, 4096, 2)
    x = rand((m, k), BF, 3)
    want = mx4.linear(x, w)
    assert want.isfinite().all()
    for rows in (1, 16, 32, 4096):
        nan = torch.full((rows, 4096), float("nan"), dtype=BF, device="cuda")
        assert mx4.linear(nan, big).isnan().all()
        assert torch.equal(mx4.linear(x, w), want)
