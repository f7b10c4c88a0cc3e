"""The gated feed-forward block's inner values: held wide by default, rounded to x's type where the caller asks for it.

Wide, an inner value h is the sum of two bf16 numbers: the nearest one and the nearest one to what is left, at most 2^-8 |h|.  A bf16
rounding is off by 2^-8 of its value, so the two are off by 2^-16 |h|, and each is a term of the second product: twice the
terms, of (1 + 2^-8) times the absolute sum.  The rest of the bound is that of the linear layers and of the gated block
(``test_gpu_mx4``); the output is rounded once.
"""

import pytest
import torch

import t2w_amd  # noqa: F401
from t2w_amd import mx4
from test_gpu_mx4 import BF, FP, U, act_of, gated_reference, rand, random_weight, rounding

pytestmark = pytest.mark.gpu


def reference(x, vg, vu, vd, act, residual=None):
    """The block in float64 and the bound of its wide form."""
    h, th = gated_reference(x, vg, vu, act)
    th = th + 2.0 ** -16 * (h.abs() + th)
    size = (h.abs() + th) * (1 + 2.0 ** -8)
    y = h @ vd.T
    tol = th @ vd.abs().T + 2 * vd.shape[1] * U * (size @ vd.abs().T)
    if residual is not None:
        y = y + residual.double()
        tol = tol + U * (y.abs() + tol)
    return y, tol + rounding(y.abs() + tol, x.dtype)


def matrices(hidden, inner, out=None):
    return random_weight(inner, hidden, 1), random_weight(inner, hidden, 2), random_weight(out or hidden, inner, 3)


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dt", [BF, FP], ids=str)
@pytest.mark.parametrize("m,hidden,inner", [(1, 256, 704), (3, 512, 1368), (8, 264, 520), (9, 264, 520), (16, 128, 8), (17, 520, 264), (50, 264, 1000), (130, 256, 520), (300, 640, 1048)])
def test_wide(dev, m, hidden, inner, dt, act):
    (g, vg), (u, vu), (d, vd) = matrices(hidden, inner)
    x, res = rand((m, hidden), dt, m), rand((m, hidden), dt, m + 1)
    y, tol = reference(x, vg, vu, vd, act, res)
    got = mx4.ffn(x, g, u, d, act=act, residual=res)
    assert got.dtype == dt and ((got.double() - y).abs() <= tol).all()


@pytest.mark.parametrize("dt", [BF, FP], ids=str)
@pytest.mark.parametrize("m,hidden,inner", [(1, 2048, 5464), (16, 2048, 5464), (40, 1024, 4096)])
def test_no_further_from_the_block_than_its_own_rounding(dev, m, hidden, inner, dt):
    """As near to 64 bits as a value that is rounded once: with inner values of x's type the error's norm is 1.2 to 1.4 times that of
    the output's rounding alone.  The fp32 sums and the pairs move a value by far less than the rounding: 2%."""
    (g, vg), (u, vu), (d, vd) = matrices(hidden, inner)
    x = rand((m, hidden), dt, m, 8 * hidden ** -0.5)
    y = act_of(x.double() @ vg.T, "silu") * (x.double() @ vu.T) @ vd.T
    got = mx4.ffn(x, g, u, d)
    alone = (y.to(dt).double() - y).norm()
    assert (got.double() - y).norm() <= 1.02 * alone


@pytest.mark.parametrize("m", [1, 12, 70, 400])
def test_inner_values_beyond_the_type(dev, m):
    """fp16: inner values far beyond 65504 and an output within its range, as the formula has it."""
    hidden, inner = 256, 520
    (g, vg), (u, vu) = random_weight(inner, hidden, 1, 8, 10), random_weight(inner, hidden, 2, 8, 10)
    d, vd = random_weight(hidden, inner, 3, -23, -22)
    x = rand((m, hidden), FP, m)
    for act in ("silu", "gelu"):
        x_ = x
        y, tol = reference(x_, vg, vu, vd, act)
        if y.abs().max() > 60000:
            x_ = x * 2.0 ** -4
            y, tol = reference(x_, vg, vu, vd, act)
        assert (act_of(x_.double() @ vg.T, act) * (x_.double() @ vu.T)).abs().max() > 1e6 and y.abs().max() < 60000
        got = mx4.ffn(x_, g, u, d, act=act)
        assert got.isfinite().all() and ((got.double() - y).abs() <= tol).all()


@pytest.mark.parametrize("dt", [BF, FP], ids=str)
@pytest.mark.parametrize("m", [2, 20, 300])
def test_infinities_and_nan_of_the_inner_values(dev, m, dt):
    """Infinite inner values give infinite outputs where the codes are not zero, NaN where they are, as the formula; the other rows keep theirs."""
    hidden, inner = 264, 520
    (g, vg), (u, vu), (d, vd) = matrices(hidden, inner)
    x = rand((m, hidden), dt, m)
    want = mx4.ffn(x, g, u, d)
    x[1, 0] = float("nan")
    x[0] = 0
    x[0, 3] = float("inf")
    got = mx4.ffn(x, g, u, d)
    assert torch.equal(got[2:], want[2:]) and got[1].isnan().all()
    h = act_of(x[:1].double() @ vg.T, "silu") * (x[:1].double() @ vu.T)
    y = (h[:, None, :] * vd[None]).sum(-1)[0]
    assert torch.equal(got[0].double().nan_to_num(nan=7.0), y.nan_to_num(nan=7.0))


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dt", [BF, FP], ids=str)
@pytest.mark.parametrize("m,hidden,inner", [(1, 256, 704), (16, 128, 8), (50, 264, 1000), (300, 640, 1048)])
def test_rounded(dev, m, hidden, inner, dt, act):
    """The caller's choice: the block's two products as calls of their own, with inner values of x's type."""
    (g, _), (u, _), (d, _) = matrices(hidden, inner)
    x, res = rand((m, hidden), dt, m), rand((m, hidden), dt, m + 1)
    got = mx4.ffn(x, g, u, d, act=act, residual=res, inner="rounded")
    assert torch.equal(got, mx4.linear(mx4.gated(x, g, u, act=act), d, residual=res))


@pytest.mark.parametrize("inner", ["wide", "rounded"])
@pytest.mark.parametrize("dt", [BF, FP], ids=str)
@pytest.mark.parametrize("m,out", [(1, 131), (8, 130), (30, 131), (300, 258)])
def test_odd_outputs(dev, m, out, dt, inner):
    """Outputs at odd strides and offsets, the residual in their place, nothing written beside them."""
    (g, vg), (u, vu), (d, vd) = matrices(264, 520, out)
    x = rand((m, 264), dt, m)
    for pad, first in ((0, 0), (7, 3), (6, 2)):
        buf = rand((m + 2, out + pad), dt, 5)
        keep, res = buf.clone(), buf[1:m + 1, first:first + out].clone()
        got = mx4.ffn(x, g, u, d, residual=buf[1:m + 1, first:first + out], out=buf[1:m + 1, first:first + out], inner=inner)
        if inner == "wide":
            y, tol = reference(x, vg, vu, vd, "silu", res)
            assert ((got.double() - y).abs() <= tol).all()
        assert torch.equal(got, mx4.ffn(x, g, u, d, residual=res, inner=inner))
        keep[1:m + 1, first:first + out] = got
        assert torch.equal(buf, keep)
