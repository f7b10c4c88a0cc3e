"""The operators of a decoder layer around the paged 8-bit cache as measurable cases: products with 4-bit weights, the gated
feed-forward block on such weights, and rotary positions of several axes.

A 4-bit weight matrix [N, K] comes as ``codes`` uint8 [N, K / 2], two e2m1 codes a byte (the lower nibble is the even column), and
``scales`` uint8 [N, ceil(K / 32)], the power of two (exponent + 127) of every 32 consecutive columns.  A code is a sign and one of
0, 0.5, 1, 1.5, 2, 3, 4, 6.

``own`` false: elementary torch operations in 32 bits.  ``own`` true: the framework's kernels (``t2w_amd.mx4``, ``t2w_amd.rope``).
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
GROUP = 32
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# --- the cases --------------------------------------------------------------------------------------------------------

def _linear(rows, n, k, dtype, bias=False, residual=False):
    return {"op": "linear", "rows": rows, "n": n, "k": k, "dtype": dtype, "bias": bias, "residual": residual}


def _ffn(rows, hidden, inner, dtype, act="silu", residual=True):
    return {"op": "ffn", "rows": rows, "hidden": hidden, "inner": inner, "dtype": dtype, "act": act, "residual": residual}


def _rope(rows, heads, kv_heads, dim, dtype, axes, pairs, form, far, rot=0):
    """``rot``: rotated channels of a head (0: all).  ``form``: ``step`` one token a row, each at a place of its own, ``grid``
    the patches of images or video frames behind a text."""
    return {"op": "rope", "rows": rows, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "axes": axes, "pairs": pairs,
            "form": form, "far": far, "rot": rot or dim}


def listed():
    return [
        # a generation step of one request: queries, keys and values of 32 over 8 heads of 128 (latency)
        dict(_linear(1, 6144, 4096, "bf16", bias=True), name="linear_step_1"),
        # the output projection of a 50-frame window in the estimator's width
        dict(_linear(50, 1024, 1024, "bf16", bias=True, residual=True), name="linear_window_50"),
        # a step of 64 requests
        dict(_linear(64, 6144, 4096, "fp16"), name="linear_step_64"),
        # the logits of three requests over an odd vocabulary
        dict(_linear(3, 128001, 4096, "bf16"), name="linear_logits_3"),
        # a chunk of prompts
        dict(_linear(4001, 6144, 4096, "bf16"), name="linear_prompt_4001"),
        # the block of a generation step of one request
        dict(_ffn(1, 4096, 14336, "bf16"), name="ffn_step_1"),
        # a step of 16 requests in a small model, inner size no multiple of the tiles
        dict(_ffn(16, 2048, 5464, "fp16", "gelu"), name="ffn_step_16"),
        # a mid-size batch: draft checks and short prompts
        dict(_ffn(200, 4096, 14336, "fp16"), name="ffn_batch_200"),
        # prompts
        dict(_ffn(2005, 4096, 14336, "bf16"), name="ffn_prompt_2005"),
        # a generation step of 64 requests at three-axis positions
        dict(_rope(64, 32, 8, 128, "bf16", 3, "halves", "step", 100000), name="rope_step_64"),
        # windows in the estimator's layout, neighbouring channels, positions of a stream that ran for hours
        dict(_rope(1608, 16, 16, 64, "bf16", 1, "neighbours", "step", 2000000000), name="rope_window_1608"),
        # a video prompt
        dict(_rope(37433, 32, 8, 128, "fp16", 3, "halves", "grid", 5000), name="rope_video_37433"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = ((16, 16, 64), (8, 8, 64), (32, 8, 128), (28, 4, 128), (16, 2, 128), (12, 4, 64), (10, 10, 128), (16, 8, 256))


def draw(rng):
    op = rng.choice(("linear", "linear", "ffn", "ffn", "rope"))
    dt = rng.choice(("bf16", "fp16"))
    if op == "rope":
        h, g, d = rng.choice(HEADS)
        form = rng.choice(("step", "grid"))
        rows = _log(rng, 1, 2000) if form == "step" else _log(rng, 100, 37000 * 40 * 128 // ((h + g) * d))
        return _rope(rows, h, g, d, dt, rng.choice((1, 2, 3, 3)), rng.choice(("halves", "halves", "neighbours")), form,
                     _log(rng, 100, 2000000000), rng.choice((0, 0, d // 2)))
    form = rng.choice(("step", "batch", "prompt"))
    rows = _log(rng, 1, 16) if form == "step" else _log(rng, 16, 300) if form == "batch" else _log(rng, 300, 4000)
    if op == "linear":
        n, k = _log(rng, 100, 40000), 8 * _log(rng, 32, 2048)
        n = max(100, min(n, 520000000 // k, 100000000000 // (rows * k)))
        return _linear(rows, n, k, dt, rng.random() < 0.5, rng.random() < 0.5)
    hidden, inner = 32 * _log(rng, 8, 160), 8 * _log(rng, 64, 2000)
    inner = max(512, min(inner, 117000000000 // (rows * hidden) // 8 * 8))
    return _ffn(rows, hidden, inner, dt, rng.choice(("silu", "silu", "gelu")), rng.random() < 0.7)


# --- what a user's program has in hand ----------------------------------------------------------------------------------

def _e2m1(x):
    """Codes of |x| <= 6, rounded to nearest, ties to the even code."""
    a = x.abs()
    c = torch.zeros(x.shape, dtype=torch.uint8, device=x.device)
    for i, edge in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)):  # a tie goes up where the code above is even
        c += (a >= edge) if i % 2 else (a > edge)
    return c | torch.where(x < 0, 8, 0).to(torch.uint8)


def _weight(n, k, gen):
    """A projection's weights, each output channel of a size of its own, in 4 bits: the scale of a group is the smallest power of
    two that keeps its largest magnitude within 6."""
    groups = -(-k // GROUP)
    w = torch.zeros(n, groups * GROUP, device=DEV)
    w[:, :k] = torch.randn(n, k, generator=gen, device=DEV)
    w *= k ** -0.5 * torch.exp2(torch.rand(n, 1, generator=gen, device=DEV) * 2 - 1)
    w = w.view(n, groups, GROUP)
    m, e = torch.frexp(w.abs().amax(-1))  # amax = m 2^e, 0.5 <= m < 1
    e = (e - 3 + (m > 0.75)).clamp(-23, 13)
    c = _e2m1(torch.ldexp(w, -e[..., None])).view(n, -1)[:, :k]
    return {"codes": (c[:, 0::2] | (c[:, 1::2] << 4)).contiguous(), "scales": (e + 127).to(torch.uint8).contiguous()}


def _axes(axes, pairs):
    """Axis of every pair: time has a quarter, the rest is split; of two axes each has half."""
    if axes == 1:
        return [0] * pairs
    if axes == 2:
        return [p * 2 // pairs for p in range(pairs)]
    t = pairs // 4
    h = (pairs - t) // 2
    return [0] * t + [1] * h + [2] * (pairs - t - h)


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device=DEV).to(TYPES[c["dtype"]])  # noqa: E731
    s = {"op": c["op"]}
    if c["op"] == "linear":
        s |= {"x": rand(c["rows"], c["k"]), "weight": _weight(c["n"], c["k"], gen)}
        s["bias"] = torch.randn(c["n"], generator=gen, device=DEV) if c["bias"] else None
        s["residual"] = rand(c["rows"], c["n"]) if c["residual"] else None
        return s
    if c["op"] == "ffn":
        s |= {"act": c["act"], "x": rand(c["rows"], c["hidden"])}
        s |= {"gate": _weight(c["inner"], c["hidden"], gen), "up": _weight(c["inner"], c["hidden"], gen), "down": _weight(c["hidden"], c["inner"], gen)}
        s["residual"] = rand(c["rows"], c["hidden"]) if c["residual"] else None
        return s
    n, h, g, d, a = c["rows"], c["heads"], c["kv_heads"], c["dim"], c["axes"]
    qkv = rand(n, h + 2 * g, d)  # queries, keys and values come as one projection's rows
    i = torch.arange(n, device=DEV)
    if c["form"] == "step":
        pos = torch.randint(0, c["far"], (1, n), generator=gen, device=DEV).expand(a, n)
    else:
        side, text = 24, 40  # patches behind the first tokens: (frame, row, column), text counts on all axes alike
        start = int(torch.randint(0, c["far"], (1,), generator=gen, device=DEV))
        j = (i - text).clamp(min=0)
        grid = (j // (side * side), j // side % side, j % side)[3 - a:]
        pos = torch.stack([torch.where(i < text, start + i, start + text + p) for p in grid])
    inv = [10000.0 ** (-2.0 * p / c["rot"]) for p in range(c["rot"] // 2)]
    s |= {"q": qkv[:, :h], "k": qkv[:, h:h + g], "pos": pos.int().contiguous(), "inv_freq": inv, "axis": _axes(a, c["rot"] // 2), "pairs": c["pairs"],
          "inv_dev": torch.tensor(inv, dtype=torch.float64, device=DEV), "axis_dev": torch.tensor(_axes(a, c["rot"] // 2), device=DEV),
          "q_out": torch.empty(n, h, d, dtype=qkv.dtype, device=DEV), "k_out": torch.empty(n, g, d, dtype=qkv.dtype, device=DEV)}
    return s


# --- the plain forms ------------------------------------------------------------------------------------------------------

def _values(w):
    """What the codes and scales stand for, fp32 [N, K]."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=DEV)
    codes = w["codes"]
    n, half = codes.shape
    v = torch.stack([table[(codes & 15).int()], table[(codes >> 4).int()]], -1).view(n, 2 * half)
    scale = torch.exp2(w["scales"].float() - 127)
    if 2 * half % GROUP == 0:
        v.view(n, -1, GROUP).mul_(scale[..., None])
    else:
        v.mul_(scale.repeat_interleave(GROUP, 1)[:, :2 * half])
    return v


def _plain_linear(x, w, bias, residual):
    y = torch.matmul(x, _values(w).T)
    if bias is not None:
        y += bias
    if residual is not None:
        y += residual.float()
    return y


def _plain_ffn(s):
    x = s["x"].float()
    a = torch.matmul(x, _values(s["gate"]).T)
    if s["act"] == "silu":
        a = a / (1 + torch.exp(-a))
    else:
        a = 0.5 * a * (1 + torch.tanh(math.sqrt(2 / math.pi) * (a + 0.044715 * a * a * a)))
    h = a * torch.matmul(x, _values(s["up"]).T)
    return _plain_linear(h, s["down"], None, s["residual"]).to(s["x"].dtype)


def _plain_rope(s):
    angle = s["pos"].double().T[:, s["axis_dev"]] * s["inv_dev"]  # [n, pairs]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    r = 2 * cos.shape[-1]
    out = {}
    for name in ("q", "k"):
        x, y = s[name].float(), s[name + "_out"]
        if s["pairs"] == "halves":
            x0, x1 = x[..., :r // 2], x[..., r // 2:r]
            turned = torch.cat([x0 * cos - x1 * sin, x0 * sin + x1 * cos], -1)
        else:
            x0, x1 = x[..., 0:r:2], x[..., 1:r:2]
            turned = torch.stack([x0 * cos - x1 * sin, x0 * sin + x1 * cos], -1).flatten(-2)
        y[..., :r] = turned
        y[..., r:] = x[..., r:]
        out[name] = y
    return out


# --- one pass ------------------------------------------------------------------------------------------------------------

def _own_weight(s, name):
    """The framework's handle of a weight: a user's program makes it once, when it loads the model."""
    from t2w_amd import mx4
    w = s.get(name + "_own")
    if w is None:
        w = s[name + "_own"] = mx4.MX4Weight(s[name]["codes"], s[name]["scales"])
    return w


def run(s):
    if own:
        import t2w_amd  # noqa: F401
        if s["op"] == "linear":
            from t2w_amd import mx4
            return mx4.linear(s["x"], _own_weight(s, "weight"), bias=s["bias"], residual=s["residual"])
        if s["op"] == "ffn":
            from t2w_amd import mx4
            return mx4.ffn(s["x"], _own_weight(s, "gate"), _own_weight(s, "up"), _own_weight(s, "down"), act=s["act"], residual=s["residual"])
        from t2w_amd import rope
        table = s.get("table")
        if table is None:  # made once with the model
            table = s["table"] = rope.Rope(s["inv_freq"], axis=s["axis"], pairs=s["pairs"], device=DEV)
        table.apply(s["q"], s["k"], s["pos"], q_out=s["q_out"], k_out=s["k_out"])
        return {"q": s["q_out"], "k": s["k_out"]}
    if s["op"] == "linear":
        return _plain_linear(s["x"].float(), s["weight"], s["bias"], s["residual"]).to(s["x"].dtype)
    return _plain_ffn(s) if s["op"] == "ffn" else _plain_rope(s)


def _weight_bytes(n, k):
    return n * k / 2 + n * -(-k // GROUP)


def work(case):
    c = dict(case)
    m = c["rows"]
    if c["op"] == "linear":
        n, k = c["n"], c["k"]
        return {"bytes": _weight_bytes(n, k) + 2.0 * m * k + 2.0 * m * n * (1 + c["residual"]) + 4.0 * n * c["bias"], "flops": 2.0 * m * n * k}
    if c["op"] == "ffn":
        h, f = c["hidden"], c["inner"]
        return {"bytes": 2 * _weight_bytes(f, h) + _weight_bytes(h, f) + 2.0 * m * h * (2 + c["residual"]), "flops": 6.0 * m * h * f}
    return {"bytes": 4.0 * m * (c["heads"] + c["kv_heads"]) * c["dim"] + 4.0 * c["axes"] * m, "flops": 3.0 * m * (c["heads"] + c["kv_heads"]) * c["rot"]}


# --- from the definition, in 64 bits ----------------------------------------------------------------------------------------

def _exact_values(w):
    """Sign, two exponent bits (bias 1) and one mantissa bit of each code, times 2 to the group's exponent."""
    nib = torch.empty(w["codes"].shape[0], 2 * w["codes"].shape[1], dtype=torch.uint8, device=DEV)
    nib[:, 0::2], nib[:, 1::2] = w["codes"] % 16, w["codes"] // 16
    e, m = (nib // 2 % 4).double(), (nib % 2).double()
    mag = torch.where(e == 0, m / 2, (1 + m / 2) * 2 ** (e - 1))
    mag = torch.where(nib >= 8, -mag, mag)
    col = torch.arange(nib.shape[1], device=DEV) // GROUP
    return mag * (2.0 ** (w["scales"].double() - 127))[:, col]


def _exact_product(x, w, step=16384):
    """x W^T over slices of W's rows."""
    n = w["codes"].shape[0]
    return torch.cat([x @ _exact_values({"codes": w["codes"][a:a + step], "scales": w["scales"][a:a + step]}).T for a in range(0, n, step)], 1)


def exact(case, seed):
    c = dict(case)
    s = prepare(case, seed)
    if c["op"] == "linear":
        y = _exact_product(s["x"].double(), s["weight"])
        y = y if s["bias"] is None else y + s["bias"].double()
        return y if s["residual"] is None else y + s["residual"].double()
    if c["op"] == "ffn":
        x = s["x"].double()
        a = _exact_product(x, s["gate"])
        a = a * torch.sigmoid(a) if c["act"] == "silu" else torch.nn.functional.gelu(a, approximate="tanh")
        y = _exact_product(a * _exact_product(x, s["up"]), s["down"])
        return y if s["residual"] is None else y + s["residual"].double()
    r = c["rot"]
    turn = torch.polar(torch.ones(1, dtype=torch.float64, device=DEV),
                       torch.stack([s["pos"][a].double() * f for a, f in zip(s["axis"], s["inv_freq"])], -1))[:, None]
    out = {}
    for name in ("q", "k"):
        x = s[name].double()
        z = torch.complex(x[..., :r // 2], x[..., r // 2:r]) if c["pairs"] == "halves" else torch.complex(x[..., 0:r:2], x[..., 1:r:2])
        z = z * turn
        y = x.clone()
        if c["pairs"] == "halves":
            y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
        else:
            y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
        out[name] = y
    return out
