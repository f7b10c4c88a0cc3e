"""The paged 8-bit cache without a GPU: what its calls refuse, the page format against the oracle, the plan's layout."""

import ctypes as C

import numpy as np
import pytest
import torch

import t2w_amd  # noqa: F401
from oracle import kv8 as ok
from t2w_amd import _lib, kv8


def pages(nb=4, g=2, d=64):
    return kv8.KV8Pages.empty(nb, g, d, device="cpu")


def ints(*v):
    return torch.tensor(v, dtype=torch.int32)


# --- the C ABI: arguments that name no memory (every call here is refused before a launch) ---

def c_pages(**kw):
    p = _lib.KV8Pages(1 << 20, 1 << 20, 1 << 20, 1 << 20, 64, 8, 128)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def refused(fn, args, text):
    assert fn(C.byref(args), None) == 1
    assert text in _lib.lib().t2w_last_error().decode()


def set_all(a, kw):
    for k, v in kw.items():
        setattr(a.pages if k in ("k_exp", "n_blocks", "kv_heads", "head_dim") else a, k, v)
    return a


PLAN_BAD = [({"n_rows": -1}, "n_rows"), ({"n_rows": 4097}, "n_rows"), ({"width": 0}, "width"), ({"ld_table": 3}, "width"), ({"n_tok": -1}, "negative"),
            ({"n_free": -1}, "negative"), ({"kv_len": None}, "null"), ({"table": None}, "null"), ({"status": None}, "null"), ({"slots": None}, "null"),
            ({"free_head_out": 3 << 20}, "output lies on an input"), ({"kv_total": 1 << 20}, "output lies on an input"),
            ({"row_start": (2 << 20) + 12}, "output lies on an input"), ({"slots": (5 << 20) + 60}, "output lies on an input"), ({"table": (1 << 20) - 60}, "table lies on an input"),
            ({"status": (4 << 20) + 60}, "output lies on the table")]


@pytest.mark.parametrize("kw,text", PLAN_BAD, ids=str)
def test_plan_refuses(kw, text):
    a = _lib.KV8PlanArgs(kv_len=1 << 20, new_len=2 << 20, n_rows=4, table=4 << 20, width=4, ld_table=4, free_ids=5 << 20, n_free=16, free_head=3 << 20,
                         n_tok=8, kv_total=6 << 20, row_start=7 << 20, tok_row=8 << 20, tok_pos=9 << 20, slots=10 << 20, free_head_out=11 << 20,
                         status=12 << 20)
    for k, v in kw.items():
        setattr(a, k, v)
    refused(_lib.lib().t2w_kv8_plan, a, text)


PAGES_BAD = [({"k_exp": None}, "null pages"), ({"head_dim": 96}, "head_dim"), ({"kv_heads": 0}, "kv_heads"), ({"n_blocks": 0}, "n_blocks"),
             ({"n_blocks": (1 << 26) + 1}, "n_blocks"), ({"n_rows": 4097}, "n_rows"), ({"width": 5}, "width"), ({"width": 1 << 26, "ld_table": 1 << 26}, "width"),
             ({"dtype": 2}, "dtype"), ({"n_tok": -1}, "negative"), ({"max_new": -1}, "negative"), ({"table": None}, "null operand")]


@pytest.mark.parametrize("kw,text", PAGES_BAD + [({"k": None}, "null operand"), ({"ldk": 1016}, "overlap"), ({"ldv": 1028}, "strides"),
                                                 ({"v": (1 << 20) + 8}, "aligned")], ids=str)
def test_append_refuses(kw, text):
    a = _lib.KV8AppendArgs(c_pages(), 1 << 20, 1 << 20, 1024, 1024, 0, 4, 1 << 20, 4, 4, 1 << 20, 1 << 20, 4, 0)
    refused(_lib.lib().t2w_kv8_append, set_all(a, kw), text)


@pytest.mark.parametrize("kw,text", PAGES_BAD + [({"out": None}, "null operand"), ({"heads": 12}, "heads"), ({"heads": 136}, "heads"), ({"heads": 0}, "heads"), ({"n_tok": (1 << 24) + 1}, "2^24"),
                                                 ({"chunk": -1}, "negative"), ({"max_kv": -5}, "negative"), ({"scale": 0.0}, "scale"),
                                                 ({"scale": float("nan")}, "scale"), ({"scale": float("inf")}, "scale"), ({"ldq": 4088}, "overlap"),
                                                 ({"ldo": 4100}, "strides"), ({"q": (1 << 20) + 2}, "aligned")], ids=str)
def test_attention_refuses(kw, text):
    a = _lib.KV8AttentionArgs(c_pages(), 1 << 20, 1 << 20, 4096, 4096, 0, 4, 32, 1 << 20, 4, 4, 1 << 20, 1 << 20, 4, 1, 0.1, 0, 0, 1 << 20, 1 << 40)
    refused(_lib.lib().t2w_kv8_attention, set_all(a, kw), text)


def test_calls_without_tokens_do_nothing():
    a = _lib.KV8AppendArgs(c_pages(), None, None, 0, 0, 0, 0, None, 4, 4, None, None, 0, 0)
    assert _lib.lib().t2w_kv8_append(C.byref(a), None) == 0
    b = _lib.KV8AttentionArgs(c_pages(), None, None, 0, 0, 0, 0, 32, None, 4, 4, None, None, 0, 1, 0.1, 0, 0, None, 0)
    assert _lib.lib().t2w_kv8_attention(C.byref(b), None) == 0
    assert _lib.lib().t2w_kv8_attention_workspace_bytes(C.byref(b)) == 0


# --- the Python calls ---

def test_pages_refuse():
    p = pages()
    with pytest.raises(ValueError, match="differ"):
        kv8.KV8Pages(p.k, p.v, p.k_exp[:3], p.v_exp)
    with pytest.raises(ValueError, match="differ"):
        kv8.KV8Pages(p.k, p.v[:, :, :, :16], p.k_exp, p.v_exp)
    with pytest.raises(ValueError, match="uint8"):
        kv8.KV8Pages(p.k.to(torch.int8), p.v, p.k_exp, p.v_exp)
    with pytest.raises(ValueError, match="uint8"):
        kv8.KV8Pages(p.k[::2], p.v[::2], p.k_exp[::2], p.v_exp[::2])
    with pytest.raises(ValueError, match="k is"):
        kv8.KV8Pages(p.k.flatten(2), p.v, p.k_exp, p.v_exp)
    with pytest.raises(ValueError, match="head_dim"):
        kv8.KV8Pages.empty(4, 2, 96, device="cpu")


def test_plan_object():
    with pytest.raises(ValueError):
        kv8.KV8Plan(4097, 8, device="cpu")
    with pytest.raises(ValueError):
        kv8.KV8Plan(4, -1, device="cpu")
    p = kv8.KV8Plan(5, 9, device="cpu")
    out = [p.kv_total, p.row_start, p.tok_row, p.tok_pos, p.slots, p.free_head, p.status]
    assert [t.numel() for t in out] == [5, 6, 9, 9, 9, 1, 1]
    spans = sorted((t.data_ptr(), t.data_ptr() + 4 * t.numel()) for t in out)
    assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:])) and all(t.data_ptr() % 16 == 0 for t in out)
    t = torch.zeros(5, 4, dtype=torch.int32)
    good = (ints(1, 2, 3, 4, 5), ints(1, 1, 1, 1, 1), t, ints(1, 2, 3), ints(0))
    for i, bad in ((0, ints(1, 2)), (1, good[1].long()), (2, t.T.contiguous().T), (2, t.long()), (3, ints(1, 2, 3, 4)[::2]), (4, ints(0, 1))):
        with pytest.raises(ValueError):
            p.build(*good[:i], bad, *good[i + 1:])
    with pytest.raises(ValueError, match="GPU"):
        p.build(*good)
    p.status.fill_(10)
    with pytest.raises(RuntimeError, match="more tokens than.*too few free"):
        p.check()
    p.status.zero_()
    p.check()


def test_append_and_attention_refuse():
    p, t = pages(), torch.zeros(2, 3, dtype=torch.int32)
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    rows = (t, ints(0, 2, 4), ints(2, 2))
    q = torch.zeros(4, 8, 64, dtype=torch.bfloat16)
    for k, v in ((x.float(), x.float()), (x, x.half()), (x, x[:3]), (x[:, :1], x[:, :1]), (x[..., :32], x[..., :32]), (x.transpose(0, 1), x), (x, x[0])):
        with pytest.raises(ValueError):
            kv8.append(p, k, v, *rows)
    with pytest.raises(ValueError):
        kv8.append(p, x, x, t, ints(0, 2), ints(2, 2))
    with pytest.raises(ValueError, match="GPU"):
        kv8.append(p, x, x, *rows)
    for bad in (q.float(), q[..., :32], q[0]):
        with pytest.raises(ValueError):
            kv8.attention(bad, p, *rows, scale=0.1)
    for out in (torch.zeros_like(q, dtype=torch.float16), q[:3].clone(), q[:, :4].clone()):
        with pytest.raises(ValueError):
            kv8.attention(q, p, *rows, scale=0.1, out=out)
    for kw in ({"max_new": 1 << 32}, {"max_kv": 1 << 31}, {"chunk": (1 << 32) + 1}):
        with pytest.raises(ValueError, match="2\\^31"):
            kv8.attention(q, p, *rows, scale=0.1, **kw)
    with pytest.raises(ValueError, match="2\\^31"):
        kv8.append(p, x, x, *rows, max_new=1 << 32)
    with pytest.raises(ValueError, match="GPU"):
        kv8.attention(q, p, *rows, scale=0.1)


@pytest.mark.parametrize("d", [64, 128])
def test_page_format(d):
    """``values`` against the byte offsets that the header states."""
    g = np.random.default_rng(d)
    p = pages(3, 2, d)
    p.k.copy_(torch.from_numpy(g.integers(0, 127, p.k.shape, dtype=np.uint8)))
    p.v.copy_(torch.from_numpy(g.integers(128, 255, p.v.shape, dtype=np.uint8)))
    p.k_exp.copy_(torch.from_numpy(g.integers(100, 140, p.k_exp.shape, dtype=np.uint8)))
    p.v_exp.copy_(torch.from_numpy(g.integers(100, 140, p.v_exp.shape, dtype=np.uint8)))
    k, v = p.values()
    k2, v2 = p.values(torch.tensor([2, 0]))
    assert torch.equal(k2, k[[2, 0]]) and torch.equal(v2, v[[2, 0]])
    kb, vb = p.k.flatten(2), p.v.flatten(2)
    for b, h, t, c in g.integers(0, [3, 2, 32, d], (200, 4)):
        ck = kb[b, h, (c // 16) * 512 + t * 16 + c % 16].view(torch.float8_e4m3fn).item()
        cv = vb[b, h, (t // 8) * 8 * d + (c // 2) * 16 + (c % 2) * 8 + t % 8].view(torch.float8_e4m3fn).item()
        assert k[b, h, t, c].item() == ck * 2.0 ** (int(p.k_exp[b, h]) - 127)
        assert v[b, h, t, c].item() == cv * 2.0 ** (int(p.v_exp[b, h]) - 127)


def test_oracle_rounding():
    """The oracle's e4m3 is torch's on every half-way and nearby value; its exponent is the smallest that fits."""
    vals = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mid = (vals[1:] + vals[:-1]) / 2
    x = torch.cat([vals, mid, mid * (1 + 1e-6), mid * (1 - 1e-6)])
    x = torch.cat([x, -x])
    assert np.array_equal(ok.e4m3(x.numpy()), x.float().to(torch.float8_e4m3fn).double().numpy())
    for a in (448.0, 449.0, 447.0, 1.0, 1.75, 1.7501, 3e38, 2.0 ** -126, 3.5 * 2.0 ** -118):
        e = ok.exponent(a)
        assert a <= 448.0 * 2.0 ** e and (e == -126 or a > 448.0 * 2.0 ** (e - 1))
    assert ok.exponent(0.0) == ok.exponent(1e-40) == -126

def attn_args(n_tok, n_rows, width, heads=32, kv_heads=8, dim=128, max_new=0, max_kv=0):
    return _lib.KV8AttentionArgs(c_pages(kv_heads=kv_heads, head_dim=dim), 1 << 20, 1 << 20, heads * dim, heads * dim, 0, n_tok, heads, 1 << 20, width,
                                 width, 1 << 20, 1 << 20, n_rows, 1, 0.1, max_new, max_kv, None, 0)


def workspace(*a, **kw):
    return _lib.lib().t2w_kv8_attention_workspace_bytes(C.byref(attn_args(*a, **kw)))


@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 8, 128), (32, 32, 128), (128, 8, 128), (1, 1, 128), (16, 16, 64), (64, 4, 64)])
def test_attention_workspace_is_bounded(heads, kv_heads, dim):
    """What a call asks for does not grow with idle rows, wide tables or missing bounds: at most 1,024 (tile, key head, part)
    of 64 packed rows, or 256 of 256."""
    most = 0
    for n_tok in (1, 4, 64, 256, 1000, 2048, 5000):
        for n_rows in (1, 2, 7, 64, 65, 256, 4096):
            for width in (1, 40, 512, 2048, 1 << 20):
                for max_new in (0, 1, 40, n_tok):
                    for max_kv in (0, 3000, 32000):
                        most = max(most, workspace(n_tok, n_rows, width, heads, kv_heads, dim, max_new, max_kv))
    assert most <= 65536 * (dim + 2) * 4


def test_steps_without_bounds_take_no_prompt_tiles():
    """64 and 256 rows of one token, no bounds, wide tables: tiles of few packed rows, whose parts need little memory."""
    assert workspace(64, 64, 2048) <= 16 << 20 and workspace(256, 256, 512) == 0
    assert workspace(64, 64, 2048, max_new=1) == 0


@pytest.mark.parametrize("rows", [1, 64, 70, 4096])
def test_a_chunk_among_resting_rows_is_split(rows):
    """256 tokens of one row over a long cache: the tile form in parts, its 256 parts of 256 packed rows, however many rows rest."""
    assert workspace(256, rows, 600, max_new=256, max_kv=16756) == 65536 * (128 + 2) * 4

def test_counts_beyond_32_bits_are_refused():
    """Sizes that the C structs' ints cannot hold: refused, not wrapped (tensors without memory stand for the large ones)."""
    big, dev = (1 << 32) + 4, torch.device("meta")
    m = lambda *s, dtype=torch.int32: torch.empty(s, dtype=dtype, device="meta")  # noqa: E731
    with pytest.raises(ValueError, match="2\\^31"):
        kv8.KV8Plan(4, 1 << 31, device="meta")
    p = kv8.KV8Pages(m(4, 2, 4, 32, 16, dtype=torch.uint8), m(4, 2, 4, 32, 2, 8, dtype=torch.uint8), m(4, 2, dtype=torch.uint8), m(4, 2, dtype=torch.uint8))
    plan = kv8.KV8Plan(2, 8, device="meta")
    with pytest.raises(ValueError, match="2\\^31"):
        plan.build(m(2), m(2), m(2, 3), m(big), m(1))
    for table in (m(2, big), m(2, big)[:, :3]):
        with pytest.raises(ValueError, match="2\\^31"):
            plan.build(m(2), m(2), table, m(8), m(1))
    x = m(big, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="2\\^31"):
        kv8.append(p, x, x, m(2, 3), m(3), m(2))
    with pytest.raises(ValueError, match="2\\^31"):
        kv8.attention(x, p, m(2, 3), m(3), m(2), scale=0.1)
    with pytest.raises(ValueError, match="2\\^31"):
        kv8.KV8Pages(m(big, 2, 4, 32, 16, dtype=torch.uint8), m(big, 2, 4, 32, 2, 8, dtype=torch.uint8), m(big, 2, dtype=torch.uint8), m(big, 2, dtype=torch.uint8))
    assert dev == plan.device
