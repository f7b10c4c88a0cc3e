"""Rotary positions of several axes on the GPU against float64, and a decoder layer of 4-bit products, positions and the 8-bit cache.

Bound of an output s (x0 cos - x1 sin): the angle's fixed point is off by 2^-32 turns and its fp32 value by half an ulp of at
most half a turn (pi 2^-24 rad: 3.2 u with u = 2^-24), sincospi by 2 ulp (4 u), the scale, the two products and the difference round once each:
10 u |s| (|x0| + |x1|) in all, then the output's eps / 2 or half its smallest step (fp16: 2^-25).
"""

import math

import numpy as np
import pytest
import torch

import t2w_amd  # noqa: F401
from oracle import rope as orp
from t2w_amd import kv8, mx4, rope

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16
U = 2.0 ** -24


def rand(shape, dt, seed):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dt)


def freqs(rot, theta=10000.0):
    return [theta ** (-2 * p / rot) for p in range(rot // 2)]


def check(got, x, pos, r, inv, axis, pairs, scale=1.0):
    want = orp.rotate(x.double().cpu().numpy(), pos.cpu().numpy(), inv, axis, pairs, scale)
    mag = np.abs(x.double().cpu().numpy())
    half = len(inv)
    i = np.arange(half) if pairs == "halves" else 2 * np.arange(half)
    j = i + half if pairs == "halves" else i + 1
    both = np.zeros_like(mag)
    both[..., i] = both[..., j] = mag[..., i] + mag[..., j]
    tol = 10 * U * abs(scale) * both
    tol = tol + np.maximum((np.abs(want) + tol) * torch.finfo(x.dtype).eps / 2, 2.0 ** -25 if x.dtype is FP else 0)
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= tol).all(), (err - tol).max()
    assert np.array_equal(got[..., 2 * half:].double().cpu().numpy(), x[..., 2 * half:].double().cpu().numpy())


@pytest.mark.parametrize("dt", [BF, FP], ids=str)
@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
@pytest.mark.parametrize("heads,kv,d,rot", [(16, 16, 64, 64), (32, 8, 128, 128), (3, 1, 128, 64), (5, 2, 80, 80), (2, 2, 96, 96), (7, 3, 72, 48), (1, 0, 16, 16), (2, 1, 256, 256), (1, 1, 1024, 1024), (33, 1, 40, 16)])
@pytest.mark.parametrize("n", [1, 5, 300])
def test_layouts(dev, n, heads, kv, d, rot, pairs, dt):
    inv = freqs(rot)
    axis = [p % 3 for p in range(rot // 2)]
    r = rope.Rope(inv, axis=axis, pairs=pairs)
    qkv = rand((n, heads + 2 * kv, d), dt, n + d)
    q, k = qkv[:, :heads], qkv[:, heads:heads + kv] if kv else None
    pos = torch.randint(-3000, 70000, (3, n), dtype=torch.int32, device="cuda")
    qo, ko = r.apply(q, k, pos)
    check(qo, q, pos, r, inv, axis, pairs)
    assert (ko is None) == (kv == 0)
    if kv:
        check(ko, k, pos, r, inv, axis, pairs)
    keep = qkv.clone()  # in place, on slices of one projection
    r.apply(q, k, pos, q_out=q, k_out=k)
    keep[:, :heads] = qo
    if kv:
        keep[:, heads:heads + kv] = ko
    assert torch.equal(qkv, keep)


@pytest.mark.parametrize("n", [511, 512, 513, 2049, 40000])
def test_many_tokens(dev, n):
    """Around the change from a token's heads in several waves to all in one, and more tokens than waves."""
    inv, axis = freqs(64), rope.sections(8, 12, 12)
    r = rope.Rope(inv, axis=axis)
    q, k = rand((n, 9, 64), BF, 1), rand((n, 3, 64), BF, 2)
    pos = torch.randint(0, 100000, (3, n), dtype=torch.int32, device="cuda")
    qo, ko = r.apply(q, k, pos)
    at = torch.cat([torch.arange(0, 40), torch.arange(n - 40, n), torch.randint(0, n, (200,))]).cuda()
    check(qo[at], q[at], pos[:, at], r, inv, axis, "halves")
    check(ko[at], k[at], pos[:, at], r, inv, axis, "halves")
    one, _ = r.apply(q[at], None, pos[:, at].contiguous())  # a token's bits do not depend on its call
    assert torch.equal(one, qo[at])


def test_far_positions(dev):
    """Every int32 position, at frequencies from a whole turn to none, negative and zero ones among them."""
    inv = [2 * math.pi, 1.0, 0.999, -0.5, 1e-9, 0.0, 3.7, 100.0]
    r = rope.Rope(inv)
    pos = torch.tensor([0, 1, -1, 2 ** 31 - 1, -2 ** 31, 2 ** 30 + 1, 16777217, 1000003], dtype=torch.int32, device="cuda")
    q = rand((8, 2, 16), FP, 1)
    got, _ = r.apply(q, None, pos)
    check(got, q, pos[None], r, inv, [0] * 8, "halves")


@pytest.mark.parametrize("scale", [0.0, 1.37, -2.0])
def test_scale_and_axes(dev, scale):
    inv = freqs(32)
    for axes in (1, 2, 16):
        axis = [p % axes for p in range(16)]
        r = rope.Rope(inv, axis=axis, scale=scale)
        buf = torch.randint(0, 999, (axes + 1, 50), dtype=torch.int32, device="cuda")  # one axis more than the pairs count on, rows of a wider table
        q = rand((21, 4, 48), FP, 1)
        got, _ = r.apply(q, None, buf[:, 7:28])
        check(got, q, buf[:, 7:28], r, inv, axis, "halves", scale)


@pytest.mark.parametrize("n", [1, 6, 700])
def test_one_row_of_positions_for_all_axes(dev, n):
    inv, axis = freqs(64), rope.sections(8, 12, 12)
    r = rope.Rope(inv, axis=axis)
    q, k = rand((n, 5, 64), BF, 1), rand((n, 2, 64), BF, 2)
    pos = torch.randint(0, 100000, (1, n), dtype=torch.int32, device="cuda")
    got = r.apply(q, k, pos.expand(3, n))
    assert all(torch.equal(a, b) for a, b in zip(got, r.apply(q, k, pos.repeat(3, 1))))
    check(got[0], q, pos.expand(3, n), r, inv, axis, "halves")


def test_strides_and_empty_calls(dev):
    r = rope.Rope(freqs(64))
    pos = torch.arange(6, dtype=torch.int32, device="cuda")
    big = rand((8, 10, 64), BF, 1)
    out = torch.full((8, 12, 64), 7.0, dtype=BF, device="cuda")
    want, _ = r.apply(big[1:7, 2:6].contiguous(), None, pos)
    r.apply(big[1:7, 2:6], None, pos, q_out=out[1:7, 3:7])
    keep = torch.full_like(out, 7.0)
    keep[1:7, 3:7] = want
    assert torch.equal(out, keep)
    q, k = r.apply(big[:0], big[:0, :2], pos[:0])
    assert q.shape == (0, 10, 64) and k.shape == (0, 2, 64)
    q, k = r.apply(big[:6, :0], big[:6, :2], pos)
    assert q.shape == (6, 0, 64) and torch.equal(k, r.apply(big[:6, :2], None, pos)[0])
    with pytest.raises(RuntimeError, match="overlap"):
        r.apply(big[:6, :4], None, pos, q_out=big[:6, 2:6])
    with pytest.raises(RuntimeError, match="16-byte"):
        flat = torch.zeros(6 * 64 + 1, dtype=BF, device="cuda")[1:].view(6, 1, 64)
        r.apply(flat, None, pos)


def test_offsets_beyond_32_bits(dev):
    r = rope.Rope(freqs(64))
    buf = torch.zeros(600, 1 << 22, dtype=BF, device="cuda")
    q = buf[:, -128:].view(600, 2, 64)
    x = rand((600, 2, 64), BF, 1)
    q.copy_(x)
    pos = torch.arange(600, dtype=torch.int32, device="cuda")
    r.apply(q, None, pos, q_out=q)
    assert torch.equal(q, r.apply(x, None, pos)[0])


# --- a decoder layer: 4-bit products, positions, the paged 8-bit cache ----------------------------------------------------------------

class Layer:
    def __init__(self, hidden, heads, kv, d, inner, dt):
        g = torch.Generator(device="cuda").manual_seed(5)
        w = lambda n, k: mx4.MX4Weight.quantize(torch.randn(n, k, generator=g, device="cuda") * k ** -0.5)  # noqa: E731
        self.heads, self.kv, self.d, self.dt = heads, kv, d, dt
        self.qkv, self.o = w((heads + 2 * kv) * d, hidden), w(hidden, heads * d)
        self.gate, self.up, self.down = w(inner, hidden), w(inner, hidden), w(hidden, inner)
        self.bias = torch.randn((heads + 2 * kv) * d, generator=g, device="cuda") * 0.1
        self.rope = rope.Rope(freqs(d), axis=rope.sections(d // 8, d // 8, d // 4))
        self.pages = kv8.KV8Pages.empty(40, kv, d)

    def __call__(self, x, pos, plan, table, max_new, max_kv):
        qkv = mx4.linear(x, self.qkv, bias=self.bias).view(-1, self.heads + 2 * self.kv, self.d)
        q, k, v = qkv.split((self.heads, self.kv, self.kv), 1)
        self.rope.apply(q, k, pos, q_out=q, k_out=k)
        kv8.append(self.pages, k, v, table, plan.row_start, plan.kv_total, max_new=max_new)
        o = kv8.attention(q, self.pages, table, plan.row_start, plan.kv_total, scale=self.d ** -0.5, chunk=1, max_new=max_new, max_kv=max_kv)
        y = mx4.linear(o.flatten(1), self.o, residual=x)
        return mx4.ffn(y, self.gate, self.up, self.down, residual=y)

    def reference(self, x, pos, seen):
        """The layer of one row in float64 over the keys and values that the cache holds of it."""
        x = x.double()
        qkv = (x @ self.qkv.values().double().T + self.bias.double()).view(-1, self.heads + 2 * self.kv, self.d)
        inv, axis = freqs(self.d), rope.sections(self.d // 8, self.d // 8, self.d // 4)
        q = torch.from_numpy(orp.rotate(qkv[:, :self.heads].cpu().numpy(), pos.cpu().numpy(), inv, axis, "halves")).cuda()
        keys, vals = (t.repeat_interleave(self.heads // self.kv, 1) for t in seen)
        n, total = x.shape[0], keys.shape[0]
        s = torch.stack([q[:, h] @ keys[:, h].T for h in range(self.heads)]) * self.d ** -0.5
        s = s.masked_fill(torch.arange(total, device="cuda") > total - n + torch.arange(n, device="cuda")[:, None], -math.inf).softmax(-1)
        o = torch.stack([s[h] @ vals[:, h] for h in range(self.heads)], 1).flatten(1)
        y = x + o @ self.o.values().double().T
        a = y @ self.gate.values().double().T
        return y + (a * torch.sigmoid(a) * (y @ self.up.values().double().T)) @ self.down.values().double().T


@pytest.mark.parametrize("dt", [BF, FP], ids=str)
@pytest.mark.parametrize("hidden,heads,kv,d,inner", [(256, 8, 2, 64, 704), (512, 4, 4, 128, 1368)])
def test_decoder_layer(dev, hidden, heads, kv, d, inner, dt):
    """Prompts of three rows, then steps of a token each, the steps by one captured graph.  Against float64 over the cache's own
    keys and values the layer rounds six times in a row (queries before and after their turn, attention, two residual sums, the inner values), each by eps / 2
    of its size at most, and the attention's weights move by their scores' error: a score of |q| |k| / sqrt(d) about 3 for
    two roundings of q.  12 roundings' worth of the outputs' norm holds all of it."""
    layer = Layer(hidden, heads, kv, d, inner, dt)
    lens = [70, 1, 33]
    table = torch.full((3, 8), -1, dtype=torch.int32, device="cuda")
    free, head = torch.randperm(40, device="cuda").int(), torch.zeros(1, dtype=torch.int32, device="cuda")
    kv_len = torch.zeros(3, dtype=torch.int32, device="cuda")
    plan, step = kv8.KV8Plan(3, sum(lens)), kv8.KV8Plan(3, 3)

    def check_rows(x, y, pos, start, totals):
        keys, vals = (t.double() for t in layer.pages.values())
        for r in range(3):
            ids = table[r, :-(-totals[r] // 32)].long()
            seen = [t[ids].transpose(1, 2).flatten(0, 1)[:totals[r]] for t in (keys, vals)]
            want = layer.reference(x[start[r]:start[r + 1]], pos[:, start[r]:start[r + 1]], seen)
            err = (y[start[r]:start[r + 1]].double() - want).norm() / want.norm()
            assert err <= 12 * torch.finfo(dt).eps / 2, err

    plan.build(kv_len, torch.tensor(lens, dtype=torch.int32, device="cuda"), table, free, head)
    plan.check()
    x = rand((sum(lens), hidden), dt, 1)
    pos = torch.stack([plan.tok_pos, plan.tok_pos // 7, plan.tok_pos % 7]).contiguous()
    y = layer(x, pos, plan, table, max(lens), 128)
    check_rows(x, y, pos, plan.row_start.tolist(), lens)
    kv_len.copy_(plan.kv_total), head.copy_(plan.free_head)

    one = torch.ones(3, dtype=torch.int32, device="cuda")
    xs, ps = rand((3, hidden), dt, 2), torch.zeros(3, 3, dtype=torch.int32, device="cuda")

    def run():
        step.build(kv_len, one, table, free, head)
        return layer(xs, ps, step, table, 1, 256)

    saved = [t.clone() for t in (table, layer.pages.k, layer.pages.v, layer.pages.k_exp, layer.pages.v_exp)]

    def restore():
        for t, s in zip((table, layer.pages.k, layer.pages.v, layer.pages.k_exp, layer.pages.v_exp), saved):
            t.copy_(s)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    restore()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    restore()
    for i in range(4):
        xs.copy_(rand((3, hidden), dt, 10 + i))
        ps.copy_(torch.stack([kv_len, kv_len // 7, kv_len % 7]))
        saved = [t.clone() for t in (table, layer.pages.k, layer.pages.v, layer.pages.k_exp, layer.pages.v_exp)]
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        step.check()
        totals = [n + 1 + i for n in lens]
        assert step.kv_total.tolist() == totals
        check_rows(xs, got, ps, [0, 1, 2, 3], totals)
        restore()
        assert torch.equal(run(), got)  # eager, the same bits
        kv_len.copy_(step.kv_total), head.copy_(step.free_head)
