"""The paged 8-bit key/value cache on the GPU against the float64 oracle: tables, append, attention, and a run of them.

Codes, exponents and tables have to be equal: a scale is a power of two, so x / 2^e is exact and rounds the same way in
every precision.  Attention's bound per output, with u = 2^-24 (an fp32 rounding), eps / 2 the type's: the scores' fp32
dot products of D exact products are off by at most (D + 2) u times their absolute sums, the scaled score, its
difference from the maximum and exp2 add a few u times the score, and a relative error of p_j by that much moves
sum p v / sum p by at most twice that times sum p |v|; a probability rounded to 16 bits for the matrix unit is off by
2^-11 at most, the sums by another (32 + D) u at any length that the tests have; the output's own rounding is eps / 2 of it,
or half the type's smallest step (fp16: 2^-25) where it lies below the normal range, whose steps do not shrink any more.
"""

import random

import numpy as np
import pytest
import torch

import t2w_amd  # noqa: F401
from oracle import kv8 as ok
from t2w_amd import kv8

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def need(n):
    return -(-n // 32)


def host(pages):
    """Code values (not scaled) and exponents as the oracle's arrays."""
    unit = kv8.KV8Pages(pages.k, pages.v, torch.full_like(pages.k_exp, 127), torch.full_like(pages.v_exp, 127))
    k, v = unit.values()
    return (k.cpu().double().numpy(), v.cpu().double().numpy(), pages.k_exp.cpu().numpy().astype(int) - 127,
            pages.v_exp.cpu().numpy().astype(int) - 127)


def scaled(pages):
    k, v = pages.values()
    return k.cpu().double().numpy(), v.cpu().double().numpy()


def random_pages(nb, g, d, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    p = kv8.KV8Pages.empty(nb, g, d)
    for t in (p.k, p.v):
        t.copy_(torch.randn(t.shape, generator=gen, device="cuda").mul(60).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8))
    p.k_exp.copy_(torch.randint(119, 124, p.k_exp.shape, generator=gen, device="cuda"))
    p.v_exp.copy_(torch.randint(116, 126, p.v_exp.shape, generator=gen, device="cuda"))
    return p


def random_table(totals, extra, seed, spare=2):
    """A table of the rows' blocks in random order, the entries behind them invalid; the block count of the pages."""
    n = sum(need(t) for t in totals) + spare
    ids = list(range(n))
    random.Random(seed).shuffle(ids)
    width = max([need(t) for t in totals] + [1]) + extra
    t = np.full((len(totals), width), -7, np.int32)
    for r, x in enumerate(totals):
        for b in range(need(x)):
            t[r, b] = ids.pop()
    return t, n


def starts(new):
    return [0] + np.cumsum(new).tolist()


# --- tables -----------------------------------------------------------------------------------------------------------

def run_plan(kv, new, width, n_free, head, n_tok, seed=0, pad=0):
    g = np.random.default_rng(seed)
    table = g.integers(0, 5000, (len(kv), width + pad)).astype(np.int32)
    free = g.permutation(100000)[:n_free].astype(np.int32)
    want = ok.plan(kv, new, table[:, :width], free, head, n_tok)
    plan = kv8.KV8Plan(len(kv), n_tok)
    dt = torch.from_numpy(table.copy()).cuda()
    plan.build(ints(kv), ints(new), dt[:, :width], torch.from_numpy(free).cuda(), ints([head]))
    got = [plan.kv_total, plan.row_start, plan.tok_row, plan.tok_pos, plan.slots, plan.free_head[0], plan.status[0], dt[:, :width]]
    for name, a, b in zip(("kv_total", "row_start", "tok_row", "tok_pos", "slots", "free_head", "status", "table"), got, want):
        assert np.array_equal(a.cpu().numpy(), np.asarray(b)), name
    assert np.array_equal(dt[:, width:].cpu().numpy(), table[:, width:])
    return plan, want


@pytest.mark.parametrize("rows", [1, 2, 63, 64, 65, 255, 256, 257, 1000, 4096])
@pytest.mark.parametrize("most", [1, 70])
def test_plan_rows(dev, rows, most):
    rng = random.Random(rows * 7 + most)
    kv = [rng.choice((0, 1, 31, 32, 33, 64, rng.randrange(500))) for _ in range(rows)]
    new = [rng.choice((0, 1, 31, 32, 33, rng.randrange(most + 1))) if most > 1 else rng.randrange(2) for _ in range(rows)]
    blocks = sum(need(a + b) - need(a) for a, b in zip(kv, new))
    run_plan(kv, new, 20, blocks + 9, 9, sum(new) + rng.randrange(3), seed=rows, pad=rows % 3)


def test_plan_lengths(dev):
    run_plan([0], [0], 1, 0, 0, 0)
    run_plan([0], [0], 1, 0, 0, 5)
    run_plan([5], [1], 1, 0, 0, 1)
    run_plan([32], [1], 2, 1, 0, 1)
    run_plan([0, 0, 40000, 7], [0, 70001, 3, 0], 4000, 3000, 1, 70100)
    run_plan([31] * 40, [1] * 40, 1, 0, 0, 1024)  # nothing to take


@pytest.mark.parametrize("kv,new,width,n_free,head,n_tok,status", [
    ([3, -1], [1, 1], 4, 9, 0, 8, 1), ([3, 4], [1, -2], 4, 9, 0, 8, 1), ([0, 0], [5, 4], 4, 9, 0, 8, 2), ([100, 0], [29, 1], 4, 9, 0, 64, 4),
    ([0, 0], [33, 1], 4, 5, 3, 64, 8), ([0], [1], 4, 5, 6, 64, 8), ([0], [1], 4, 5, -1, 64, 8), ([-1, 0], [40, 90], 2, 0, 0, 64, 15),
    ([2 ** 31 - 1, 5], [2 ** 31 - 1, 2 ** 31 - 1], 4, 9, 0, 64, 14)], ids=str)
def test_plan_that_cannot_be_served(dev, kv, new, width, n_free, head, n_tok, status):
    """Nothing is taken, the table stays, no row has new tokens, and ``check`` says what is wrong."""
    plan, want = run_plan(kv, new, width, n_free, head, n_tok)
    assert want[6] == status
    with pytest.raises(RuntimeError, match="kv8 plan"):
        plan.check()


# --- append -------------------------------------------------------------------------------------------------------------

def check_append(pages, k, v, table, new, totals, max_new=0):
    want = host(pages)
    ok.append(*want, k.double().cpu().numpy(), v.double().cpu().numpy(), table, starts(new), totals)
    kv8.append(pages, k, v, torch.from_numpy(table).cuda(), ints(starts(new)), ints(totals), max_new=max_new)
    for name, a, b in zip(("k", "v", "k_exp", "v_exp"), host(pages), want):
        assert np.array_equal(a, b, equal_nan=True), name


def new_kv(n, g, d, dt, seed, spread=3):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    def one():
        x = torch.randn(n, g, d, generator=gen, device="cuda")
        return (x * torch.exp2(spread * torch.randn(n, 1, 1, generator=gen, device="cuda"))).to(dt)
    return one(), one()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("g", [1, 2, 5])
@pytest.mark.parametrize("bound", [0, 70, 3])
def test_append_lengths(dev, d, dt, g, bound):
    """Old and new lengths around the block's, rows without new tokens; with the longest row's length, none and one that
    is too small."""
    old = [0, 0, 1, 31, 32, 33, 40, 63, 64, 5, 17, 30]
    new = [1, 70, 1, 1, 1, 31, 0, 2, 33, 27, 64, 3]
    totals = [a + b for a, b in zip(old, new)]
    table, nb = random_table(totals, 1, seed=g)
    k, v = new_kv(sum(new), g, d, dt, seed=d + g)
    check_append(random_pages(nb, g, d, g), k, v, table, new, totals, max_new=bound)


@pytest.mark.parametrize("rows", [63, 64, 65, 300, 4096])
def test_append_many_rows(dev, rows):
    rng = random.Random(rows)
    old = [rng.randrange(40) for _ in range(rows)]
    new = [rng.choice((0, 1, 1, 2, 35)) if rows < 4096 else rng.randrange(2) for _ in range(rows)]
    totals = [a + b for a, b in zip(old, new)]
    table, nb = random_table(totals, 0, seed=1)
    k, v = new_kv(sum(new), 1, 64, BF, seed=rows)
    pages = random_pages(nb, 1, 64, 2)
    for bound in (0, max(new)):
        check_append(pages, k, v, table, new, totals, max_new=bound)  # the second time over what the first one stored


@pytest.mark.parametrize("dt", [BF, FP])
def test_append_strided_and_extremes(dev, dt):
    """Slices of a joint projection; zeros, subnormals, the type's largest values, negative zeros."""
    n, g, d = 40, 3, 64
    x = torch.randn(n, 11, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(dt)
    k, v = x[:, 4:7], x[:, 8:11]
    k[3], k[4], v[5], v[33:] = 0, torch.finfo(dt).max, torch.finfo(dt).smallest_normal / 4, 0
    k[6], v[7] = -0.0, -torch.finfo(dt).max
    old, new = [0, 7, 30], [33, 2, 5]
    totals = [a + b for a, b in zip(old, new)]
    table, nb = random_table(totals, 0, seed=3)
    check_append(random_pages(nb, g, d, 5), k, v, table, new, totals)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("factor", [2.0 ** -12, 1.0, 2.0 ** 6, 2.0 ** 40])
def test_append_rescales_the_block(dev, d, factor):
    """Token by token into one block, each step ``factor`` larger or smaller: the old codes follow the scale."""
    pages = random_pages(2, 2, d, 1)
    table = np.array([[1]], np.int32)
    for t in range(33 - 1):
        k, v = new_kv(1, 2, d, BF, seed=t)
        s = factor ** min(t, 3)
        check_append(pages, (k * s).to(BF), (v * s).to(BF), table, [1], [t + 1], max_new=1)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dt", [BF, FP])
def test_append_not_finite(dev, d, dt):
    """Infinities and NaN in keys or values, one head of them, first and last channels and tokens, a whole block."""
    old, new = [0, 9, 32], [40, 20, 3]
    totals = [a + b for a, b in zip(old, new)]
    table, nb = random_table(totals, 0, seed=2)
    k, v = new_kv(sum(new), 3, d, dt, seed=1)
    k[0, 0, 0] = float("inf")
    v[31, 1, d - 1] = float("nan")
    k[33, 2, 17], v[33, 2, 5] = float("nan"), float("-inf")
    v[45, 0, 3] = float("-inf")
    k[60:63, 1] = float("nan")
    check_append(random_pages(nb, 3, d, 4), k, v, table, new, totals)


def test_append_skips_foreign_blocks(dev):
    """Ids outside the pages and rows past their table store nothing; the others are stored."""
    old, new = [0, 3, 0], [40, 2, 33]
    totals = [a + b for a, b in zip(old, new)]
    table = np.array([[-1, 2], [5, 0], [1, 2 ** 31 - 1]], np.int32)
    k, v = new_kv(sum(new), 2, 64, BF, seed=1)
    check_append(random_pages(5, 2, 64, 1), k, v, table, new, totals)
    check_append(random_pages(5, 2, 64, 1), k, v, table, new, totals, max_new=40)
    wide = np.array([[3], [4], [1]], np.int32)  # 40 and 33 tokens in one block's width: their first 32
    pages = random_pages(5, 2, 64, 1)
    want = host(pages)
    for r, t0 in ((0, 0), (2, 42)):
        ok.append(*want, k[t0:t0 + 32].double().cpu().numpy(), v[t0:t0 + 32].double().cpu().numpy(), wide[r:r + 1], [0, 32], [32])
    ok.append(*want, k[40:42].double().cpu().numpy(), v[40:42].double().cpu().numpy(), wide[1:2], [0, 2], [5])
    kv8.append(pages, k, v, torch.from_numpy(wide).cuda(), ints(starts(new)), ints(totals))
    for a, b in zip(host(pages), want):
        assert np.array_equal(a, b)

@pytest.mark.parametrize("first", [1, 3, 70])
def test_append_rows_of_a_larger_call(dev, first):
    """The last rows of a call by slices of its tables: starts beyond the first token, nothing done before the first row.  The
    table's entries before the slice are blocks of a scale byte 0, which any second look at them would raise."""
    rows = 75
    new = [(1, 40, 0, 33)[r % 4] for r in range(rows)]
    old = [(0, 5, 32, 31)[r % 4] for r in range(rows)]
    totals = [a + b for a, b in zip(old, new)]
    table, nb = random_table(totals, 0, seed=first, spare=3)
    spare = sorted(set(range(nb)) - set(table[r, b] for r, t in enumerate(totals) for b in range(need(t))))
    for r in range(first):
        table[r, :] = spare[r % len(spare)]
    pages = random_pages(nb, 2, 64, seed=1)
    pages.k_exp[spare], pages.v_exp[spare] = 0, 0
    k, v = new_kv(sum(new), 2, 64, BF, seed=2)
    want = host(pages)
    ok.append(*want, k.double().cpu().numpy(), v.double().cpu().numpy(), table[first:], starts(new)[first:], totals[first:])
    dt = torch.from_numpy(table).cuda()
    kv8.append(pages, k, v, dt[first:], ints(starts(new))[first:], ints(totals)[first:])
    for name, a, b in zip(("k", "v", "k_exp", "v_exp"), host(pages), want):
        assert np.array_equal(a, b), name

@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dt", [BF, FP])
def test_append_to_blocks_of_foreign_scales(dev, d, dt):
    """Blocks filled elsewhere, of the scales 2^127 (byte 254), 2^-127 (0) and 2^-126 (1), go on with them or with what the new tokens
    need; one of an E8M0 NaN stays NaN."""
    old, new = [9, 9, 9, 9, 30], [3, 3, 3, 3, 9]
    totals = [a + b for a, b in zip(old, new)]
    table, nb = random_table(totals, 0, seed=1)
    k, v = new_kv(sum(new), 2, d, dt, seed=3)
    k[0], v[1] = torch.finfo(dt).max, torch.finfo(dt).max
    k[3:6] *= 0
    for heads in (slice(0, 2), slice(1, 2)):
        pages = random_pages(nb, 2, d, seed=2)
        for r, e in ((0, 254), (1, 0), (2, 1)):
            pages.k_exp[int(table[r, 0]), heads], pages.v_exp[int(table[r, 0]), heads] = e, e
        check_append(pages, k, v, table, new, totals)
    pages = random_pages(nb, 2, d, seed=2)
    pages.k_exp[int(table[3, 0]), 1] = 255
    want = host(pages)
    ok.append(*want, k.double().cpu().numpy(), v.double().cpu().numpy(), table, starts(new), totals)
    kv8.append(pages, k, v, torch.from_numpy(table).cuda(), ints(starts(new)), ints(totals))
    for i, (a, b) in enumerate(zip(host(pages), want)):
        if i == 0:  # codes under a scale of NaN stand for nothing
            a[int(table[3, 0]), 1] = b[int(table[3, 0]), 1] = 0
        assert np.array_equal(a, b)


# --- attention ------------------------------------------------------------------------------------------------------------

def attn_bound(o, mag, top, d, dt):
    u = 2.0 ** -24
    rel_p = 2 * ((d + 2) * u * top + 8 * u * (top * 1.4427 + 2) + 2.0 ** -11) + 2 * (32 + d) * u
    f = torch.finfo(dt)
    return f.eps / 2 * np.maximum(np.abs(o), f.smallest_normal) * 1.01 + rel_p[:, :, None] * mag * 1.01


def check_attention(q, pages, table, new, totals, chunk, scale=None, **kw):
    d = pages.head_dim
    scale = scale or d ** -0.5
    k, v = scaled(pages)
    o, mag, top = ok.attention(q.double().cpu().numpy(), k, v, table, starts(new), totals, scale, chunk)
    out = kv8.attention(q, pages, torch.from_numpy(table).cuda(), ints(starts(new)), ints(totals), scale=scale, chunk=chunk, **kw)
    torch.cuda.synchronize()
    n = sum(new)
    got = out[:n].double().cpu().numpy()
    bound = attn_bound(o, mag, top, d, q.dtype)[:n]
    assert np.isfinite(got).all()
    worst = float((np.abs(got - o[:n]) / bound).max()) if n else 0.0
    assert worst <= 1, worst
    return out


def queries(n, h, d, dt, seed):
    return torch.randn(n, h, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dt)


HEADS = [(1, 1), (4, 4), (16, 16), (6, 2), (8, 2), (7, 1), (14, 2), (32, 2)]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("h,g", HEADS)
def test_attention_steps(dev, d, dt, h, g):
    """One token a row, caches from that token alone to several hundred, rows without a token."""
    totals = [1, 2, 31, 32, 33, 64, 65, 200, 417, 7]
    new = [1, 1, 1, 1, 1, 1, 0, 1, 1, 0]
    table, nb = random_table(totals, 1, seed=h)
    pages = random_pages(nb, g, d, seed=d)
    q = queries(sum(new), h, d, dt, seed=g)
    for bounds in ({"max_new": 1, "max_kv": 417}, {"max_new": 1}, {}):
        check_attention(q, pages, table, new, totals, 1, **bounds)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("h,g", [(2, 2), (6, 2), (7, 1), (16, 1)])
@pytest.mark.parametrize("chunk", [0, 1, 3, 25])
def test_attention_windows(dev, d, dt, h, g, chunk):
    """Windows of several lengths behind caches of several lengths."""
    old = [0, 10, 32, 100, 63, 5, 0, 250]
    new = [1, 50, 33, 2, 64, 0, 70, 17]
    totals = [a + b for a, b in zip(old, new)]
    table, nb = random_table(totals, 0, seed=chunk)
    pages = random_pages(nb, g, d, seed=d + chunk)
    q = queries(sum(new), h, d, dt, seed=g)
    for bounds in ({"max_new": 70, "max_kv": max(totals)}, {}):
        check_attention(q, pages, table, new, totals, chunk, **bounds)


@pytest.mark.parametrize("new", [2, 4, 5, 9, 16, 17, 31])
@pytest.mark.parametrize("h,g", [(4, 4), (8, 2), (14, 2)])
def test_attention_few_tokens(dev, new, h, g):
    """A few tokens a row (drafts being checked): the packed rows of a tile around its sizes, long caches."""
    totals = [new, 300, 1500, 40 + new]
    table, nb = random_table(totals, 0, seed=new)
    pages = random_pages(nb, g, 128, seed=new)
    q = queries(4 * new, h, 128, BF, seed=g)
    check_attention(q, pages, table, [new] * 4, totals, 1, max_new=new, max_kv=1500)


@pytest.mark.parametrize("d,dt", [(64, BF), (128, FP)])
@pytest.mark.parametrize("rows,new,old", [(1, 1, 5000), (2, 3, 3000), (1, 130, 900), (1, 200, 0), (3, 129, 64)])
def test_attention_long(dev, d, dt, rows, new, old):
    """Key lists that few workgroups have to themselves: split and joined."""
    totals = [old + new - 37 * r for r in range(rows)]
    table, nb = random_table(totals, 3, seed=new)
    pages = random_pages(nb, 2, d, seed=1)
    q = queries(rows * new, 4, d, dt, seed=2)
    for chunk in (0, 1):
        for bounds in ({"max_new": new, "max_kv": max(totals)}, {"max_new": new, "max_kv": 100}, {"max_new": new, "max_kv": 1 << 20}, {}):
            check_attention(q, pages, table, [new] * rows, totals, chunk, **bounds)


# calls that the tile form takes: heads of 128, 256-row tiles mostly full, 224 workgroups or more
TILE = [(1, 32, 7, 200), (2, 32, 7, 101), (4, 16, 7, 97), (7, 16, 7, 70), (16, 14, 8, 31), (3, 29, 8, 170)]  # group, kv_heads, rows, new


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("G,g,rows,new", TILE)
@pytest.mark.parametrize("chunk", [0, 1, 7])
def test_attention_prompts(dev, dt, G, g, rows, new, chunk):
    """Many packed rows: whole prompts and prompts behind cached tokens of several lengths, some ragged."""
    new_l = [max(1, new - (5 * r if r % 3 == 1 else 0)) for r in range(rows)]
    totals = [n + (0, 1, 40, 95, 300)[r % 5] for r, n in enumerate(new_l)]
    table, nb = random_table(totals, 1, seed=G)
    pages = random_pages(nb, g, 128, seed=new)
    q = queries(sum(new_l), G * g, 128, dt, seed=g)
    check_attention(q, pages, table, new_l, totals, chunk, max_new=new, max_kv=max(totals))


@pytest.mark.parametrize("dt", [BF, FP])
def test_attention_prompt_in_parts(dev, dt):
    """A chunk of a prompt over a long cache: key lists cut so that the tiles fill the chip, block ids beyond the first 64
    of a part."""
    table, nb = random_table([17000], 1, seed=3)
    pages = random_pages(nb, 32, 128, seed=3)
    for chunk in (0, 1):
        check_attention(queries(256, 32, 128, dt, seed=4), pages, table, [256], [17000], chunk, max_new=256, max_kv=17000)


def test_attention_rows_of_many_tiles(dev):
    """More than 64 rows, of one to three tiles and none."""
    new = [(0, 1, 130, 64, 200, 65, 3)[r % 7] for r in range(80)]
    totals = [n + 9 * (r % 11) for r, n in enumerate(new)]
    table, nb = random_table(totals, 0, seed=1)
    for d, h in ((64, 1), (128, 4)):
        pages = random_pages(nb, h, d, seed=3)
        q = queries(sum(new), h, d, BF, seed=4)
        for bounds in ({"max_new": 200, "max_kv": 300}, {}):
            check_attention(q, pages, table, new, totals, 1, **bounds)


@pytest.mark.parametrize("rows", [65, 500, 4096])
def test_attention_many_rows(dev, rows):
    rng = random.Random(rows)
    new = [rng.choice((0, 1, 2)) if rows < 4096 else int(r % 64 == 5) for r in range(rows)]
    totals = [n + rng.randrange(60) for n in new]
    table, nb = random_table(totals, 0, seed=1)
    pages = random_pages(nb, 1, 64, seed=3)
    q = queries(sum(new), 2, 64, BF, seed=4)
    for bounds in ({"max_new": 2, "max_kv": 62}, {}):
        check_attention(q, pages, table, new, totals, 1, **bounds)


@pytest.mark.parametrize("new", [1, 40, 140])
def test_attention_scores_of_any_size(dev, new):
    """Large scores (one key takes all), and scores far below zero everywhere: no underflow to an empty row."""
    totals = [new + 100, new]
    table, nb = random_table(totals, 0, seed=1)
    pages = random_pages(nb, 2, 64, seed=5)
    q = queries(2 * new, 4, 64, BF, seed=6)
    check_attention(q * 16, pages, table, [new] * 2, totals, 1)
    pages.k.bitwise_and_(0x7F)  # keys of one sign, queries of the other
    check_attention(-(q.abs() * 1024).to(BF), pages, table, [new] * 2, totals, 1)
    pages.k_exp.add_(60)  # scores of 2^60 and more: the maximum alone counts
    out = kv8.attention(-q.abs(), pages, torch.from_numpy(table).cuda(), ints([0, new, 2 * new]), ints(totals), scale=1.0, chunk=1)
    assert torch.isfinite(out).all() and (out.abs().amax((1, 2)) > 0).all()


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("new", [1, 40])
def test_attention_scales_of_any_size(dev, new, dt):
    """Value scales that differ by 2^20 between blocks, growing and falling along the row."""
    totals = [new + 200, new + 90]
    table, nb = random_table(totals, 0, seed=1)
    pages = random_pages(nb, 2, 64, seed=5)
    for r in range(2):
        for b in range(need(totals[r])):
            pages.v_exp[table[r, b]] = 112 + (7 * b % 21 if r else 3 * b)
    q = queries(2 * new, 2, 64, dt, seed=6)
    check_attention(q, pages, table, [new] * 2, totals, 0)


@pytest.mark.parametrize("new", [2, 40, 140])
def test_attention_empty_rows(dev, new):
    """Rows whose cache is shorter than their queries (kv_total < new): the first ones see nothing and get zeros."""
    new_l, totals = [new, new, new], [new - 1, 0, new // 2]
    table, nb = random_table(totals, 1, seed=1)
    pages = random_pages(nb, 2, 64, seed=5)
    q = queries(3 * new, 4, 64, BF, seed=6)
    for chunk in (0, 1, 7):
        for bounds in ({"max_new": new}, {}):
            check_attention(q, pages, table, new_l, totals, chunk, **bounds)


FORMS = [(1, 4, 2, 64, 3), (40, 4, 2, 64, 3), (140, 4, 2, 64, 3), (1, 4, 2, 128, 3), (20, 4, 2, 128, 4), (40, 2, 2, 128, 3), (101, 64, 32, 128, 7)]


@pytest.mark.parametrize("new,h,g,d,rows", FORMS)
def test_attention_ignores_what_lies_behind(dev, new, h, g, d, rows):
    """NaN codes and E8M0 NaN scales behind the rows' last tokens and in blocks of nobody, ids behind the rows' tables."""
    totals = [new + (100, 11, 0)[r % 3] for r in range(rows)]
    table, nb = random_table(totals, 2, seed=1)
    pages = random_pages(nb, g, d, seed=5)
    used = sorted(x for r, t in enumerate(totals) for x in table[r, :need(t)])
    for b in set(range(nb)) - set(used):
        pages.k[b], pages.v[b], pages.k_exp[b], pages.v_exp[b] = 255, 255, 255, 255
    k, v = pages.k, pages.v
    q = queries(rows * new, h, d, BF, seed=6)
    clean = check_attention(q, pages, table, [new] * rows, totals, 1, max_new=new, max_kv=max(totals)).clone()
    for r, t in enumerate(totals):
        if t % 32:
            b = int(table[r, t // 32])
            k[b, :, :, t % 32:] = 0x7F
            vv = v[b].permute(0, 1, 4, 2, 3).reshape(g, 32, d // 2, 2).clone()
            vv[:, t % 32:] = 0xFF
            v[b] = vv.reshape(g, 4, 8, d // 2, 2).permute(0, 1, 3, 4, 2)
    for bounds in ({}, {"max_new": new}, {"max_new": new, "max_kv": max(totals)}):
        out = kv8.attention(q, pages, torch.from_numpy(table).cuda(), ints(starts([new] * rows)), ints(totals), scale=d ** -0.5, chunk=1, **bounds)
        assert torch.isfinite(out).all()
    assert torch.equal(out, clean)


@pytest.mark.parametrize("new,h,g,d,rows", FORMS)
def test_attention_nan_tokens_reach_only_who_sees_them(dev, new, h, g, d, rows):
    """A NaN key (stored by the append for a token that is not finite) in causal windows: earlier queries are untouched."""
    old = 70
    totals = [old + new] * rows
    table, nb = random_table(totals, 0, seed=1)
    pages = random_pages(nb, g, d, seed=5)
    q = queries(rows * new, h, d, BF, seed=6)
    args = (torch.from_numpy(table).cuda(), ints(starts([new] * rows)), ints(totals))
    clean = kv8.attention(q, pages, *args, scale=0.125, chunk=1, max_new=new)
    at = old + new // 2
    pages.k[int(table[0, at // 32]), 1, :, at % 32] = 0x7F
    out = kv8.attention(q, pages, *args, scale=0.125, chunk=1, max_new=new)
    hit = torch.zeros(rows * new, h, dtype=torch.bool, device="cuda")
    hit[new // 2:new, h // g:2 * (h // g)] = True
    assert out[hit].isnan().all() and torch.equal(out[~hit], clean[~hit])


@pytest.mark.parametrize("new,h,g,d,rows", FORMS)
def test_attention_malformed_rows(dev, new, h, g, d, rows):
    """Block ids outside the pages and rows longer than their table: NaN for who sees them, the others as ever.  Block 0 of
    the pages holds NaN codes, as memory that nothing was appended to may."""
    rows = max(rows, 4)
    totals = [new + 100] * rows
    table, nb = random_table(totals, 0, seed=1)
    table = np.where(table == 0, nb - 1, table) if 0 in table else table  # block 0 belongs to nobody
    pages = random_pages(nb, g, d, seed=5)
    pages.k[0], pages.v[0] = 0x7F, 0xFF
    q = queries(rows * new, h, d, BF, seed=6)
    start = ints(starts([new] * rows))
    clean = kv8.attention(q, pages, torch.from_numpy(table).cuda(), start, ints(totals), scale=0.125, chunk=1, max_new=new)
    assert torch.isfinite(clean).all()
    table[1, 1] = nb
    table[2, 0] = -1
    table[0, (totals[0] - 1) // 32] = 1 << 30  # the last new tokens' block: the tokens before it do not see it
    out = kv8.attention(q, pages, torch.from_numpy(table).cuda(), start, ints(totals[:3] + [table.shape[1] * 32 + 1] + totals[4:]), scale=0.125, chunk=1,
                        max_new=new)
    first = max(0, (totals[0] - 1) // 32 * 32 - 100)  # row 0's first token that does
    assert torch.equal(out[:first], clean[:first]) and out[first:4 * new].isnan().all() and torch.equal(out[4 * new:], clean[4 * new:])
    if new > 1:  # a row of more new tokens than the bound says: NaN where the bound chose the kernel
        out = kv8.attention(q[:new + 1], pages, torch.from_numpy(table[:2] * 0 + 1).cuda(), ints([0, new, new + 1]), ints(totals[:2]), scale=0.125, chunk=1,
                            max_new=1)
        assert (out[:new].isnan().all() or torch.isfinite(out[:new]).all()) and torch.isfinite(out[new]).all()


@pytest.mark.parametrize("new", [1, 40, 140])
def test_attention_strides_and_rows_behind(dev, new):
    """q a slice of a joint projection, out a slice of a larger buffer; rows behind the last token stay; a caller's
    workspace."""
    totals = [new + 50, new]
    table, nb = random_table(totals, 0, seed=1)
    pages = random_pages(nb, 2, 64, seed=5)
    qkv = torch.randn(2 * new + 3, 9, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(BF)
    buf = torch.full((2 * new + 3, 7, 64), 5.0, device="cuda", dtype=BF)
    ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    out = check_attention(qkv[:, 2:6], pages, table, [new] * 2, totals, 1, out=buf[:, 1:5], workspace=ws)
    assert (out[2 * new:] == 5).all() and (buf[:, 0] == 5).all() and (buf[:, 5:] == 5).all()
    again = kv8.attention(qkv[:, 2:6].contiguous(), pages, torch.from_numpy(table).cuda(), ints(starts([new] * 2)), ints(totals), scale=0.125, chunk=1)
    assert torch.equal(again[:2 * new], out[:2 * new])


def test_pages_beyond_32_bit_offsets(dev):
    """Blocks whose bytes lie beyond 4 GiB in the pages: the same codes and outputs as at the pages' start."""
    g, d, nb = 8, 128, 140000  # 32 KB a block: 4.6 GB of keys, as much of values
    dev_ = torch.device("cuda", torch.cuda.current_device())
    e = lambda *s: torch.empty(s, dtype=torch.uint8, device=dev_)  # noqa: E731
    big = kv8.KV8Pages(e(nb, g, d // 16, 32, 16), e(nb, g, 4, d // 2, 2, 8), e(nb, g), e(nb, g))
    assert big.k.numel() > 1 << 32
    for old, new, h in ((0, 70, 16), (70, 1, 16), (71, 1, 128), (72, 40, 8)):
        n = need(old + new)
        low = kv8.KV8Pages(*(t[:n] for t in (big.k, big.v, big.k_exp, big.v_exp)))
        k, v = new_kv(new, g, d, BF, seed=new)
        q = queries(new, h, d, BF, seed=old)
        outs = []
        for pages, first in ((low, 0), (big, nb - n - 1)):
            table = torch.arange(first, first + n, dtype=torch.int32, device="cuda")[None]
            if first:  # what the low blocks held before this step lies in the high ones too
                for t in (big.k, big.v, big.k_exp, big.v_exp):
                    t[first:first + n].copy_(before[t.data_ptr()])
            else:
                before = {t.data_ptr(): t[:n].clone() for t in (big.k, big.v, big.k_exp, big.v_exp)}
            args = (table, ints([0, new]), ints([old + new]))
            kv8.append(pages, k, v, *args, max_new=new)
            outs.append(kv8.attention(q, pages, *args, scale=0.1, chunk=1, max_new=new, max_kv=old + new))
        assert torch.isfinite(outs[0]).all() and torch.equal(*outs)
        for t in (big.k, big.v, big.k_exp, big.v_exp):
            assert torch.equal(t[:n], t[nb - n - 1:nb - 1])


@pytest.mark.parametrize("h,g,d,new,old", [(16, 16, 64, 1, 700), (32, 8, 128, 1, 4000), (16, 16, 64, 50, 320), (32, 8, 128, 500, 77)])
def test_attention_in_place(dev, h, g, d, new, old):
    """The outputs over the queries' own memory: the bits of the call with an output of its own (each kernel form, split or not)."""
    totals = [old + new, new, old + new + 31, old + new - 7]
    table, nb = random_table(totals, 0, seed=new)
    pages = random_pages(nb, g, d, 5)
    q = queries(4 * new, h, d, BF, seed=6)
    args = (pages, torch.from_numpy(table).cuda(), ints(starts([new] * 4)), ints(totals))
    kw = dict(scale=d ** -0.5, chunk=1, max_new=new, max_kv=max(totals))
    want = kv8.attention(q, *args, **kw)
    assert kv8.attention(q, *args, out=q, **kw) is q
    assert torch.equal(q, want)


def test_attention_same_bits_every_time(dev):
    totals = [3000, 1700, 4000, 60]
    for new in (1, 3, 60):
        table, nb = random_table(totals, 0, seed=1)
        pages = random_pages(nb, 2, 128, seed=5)
        q = queries(4 * new, 8, 128, BF, seed=6)
        args = (q, pages, torch.from_numpy(table).cuda(), ints(starts([new] * 4)), ints(totals))
        first = kv8.attention(*args, scale=0.1, chunk=1, max_new=new, max_kv=4000)
        for _ in range(5):
            assert torch.equal(kv8.attention(*args, scale=0.1, chunk=1, max_new=new, max_kv=4000), first)


def test_attention_on_other_streams(dev):
    """Two calls at once on two streams, each with the workspace it takes for itself."""
    totals = [5000, 4100]
    table, nb = random_table(totals, 0, seed=1)
    pages = random_pages(nb, 2, 128, seed=5)
    args = (pages, torch.from_numpy(table).cuda(), ints([0, 1, 2]), ints(totals))
    qs = [queries(2, 8, 128, BF, seed=s) for s in range(2)]
    want = [kv8.attention(q, *args, scale=0.1, max_new=1, max_kv=5000) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    for _ in range(10):
        got = []
        for s, q in zip(streams, qs):
            with torch.cuda.stream(s):
                got.append(kv8.attention(q, *args, scale=0.1, max_new=1, max_kv=5000))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))

@pytest.mark.parametrize("rows,n_tok,at,width,old", [(64, 64, None, 2048, 700), (200, 200, None, 512, 90), (64, 256, 5, 600, 16500), (70, 256, 69, 600, 16500),
                                                     (4096, 256, 1234, 600, 16500), (130, 400, 64, 600, 16500)])
@pytest.mark.parametrize("bounds", [False, True])
def test_attention_idle_rows_and_wide_tables(dev, rows, n_tok, at, width, old, bounds):
    """Many rows of one token and a wide table; one prompt chunk among rows that rest or have a token (32 heads over 8 of 128)."""
    new = [1] * rows if at is None else [0] * rows
    if at is not None:
        new[at] = min(n_tok, 256)
        for r in range(n_tok - new[at]):
            new[(at + 1 + r) % rows if r < rows - 1 else at] += 1
    totals = [n + (old if n > 1 else 5 * (r % 50)) if n else 0 for r, n in enumerate(new)]
    table, nb = random_table(totals, 0, seed=rows)
    table = np.concatenate([table, np.full((rows, width - table.shape[1]), -1, np.int32)], 1)
    pages = random_pages(nb, 8, 128, seed=1)
    q = queries(sum(new), 32, 128, BF, seed=2)
    check_attention(q, pages, table, new, totals, 1, **({"max_new": max(new), "max_kv": max(totals)} if bounds else {}))

# every kernel form: (new, old, heads, kv_heads, dim, rows); 16 packed rows, 32, 2 x 32, key lists in parts, the tile form, its parts
ALL_FORMS = [(1, 100, 4, 2, 64, 3), (12, 100, 4, 2, 128, 3), (40, 100, 4, 2, 64, 3), (1, 2500, 4, 2, 128, 2), (101, 60, 64, 32, 128, 7),
             (256, 14200, 32, 32, 128, 1)]


@pytest.mark.parametrize("new,old,h,g,d,rows", ALL_FORMS)
def test_attention_key_scale_byte_zero(dev, new, old, h, g, d, rows):
    """Blocks whose key scale is 2^-127, seen whole and in part: scores of (nearly) zero, not NaN.  And pages as they are made:
    zeros."""
    totals = [old + new - 13 * r for r in range(rows)]
    table, nb = random_table(totals, 0, seed=1)
    pages = random_pages(nb, g, d, seed=5)
    for r, t in enumerate(totals):
        pages.k_exp[torch.from_numpy(table[r, (need(t) - 1) % 2:need(t):2]).long().cuda()] = 0  # the last block among them
    q = queries(rows * new, h, d, BF, seed=6)
    bounds = {"max_new": new, "max_kv": max(totals)}
    check_attention(q, pages, table, [new] * rows, totals, 1, **bounds)
    check_attention(q, pages, table, [new] * rows, [t - 3 for t in totals], 7, **bounds)
    pages.k_exp.zero_()
    check_attention(q, pages, table, [new] * rows, totals, 1, **bounds)
    out = kv8.attention(q, kv8.KV8Pages.empty(nb, g, d), torch.from_numpy(table).cuda(), ints(starts([new] * rows)), ints(totals), scale=0.1, chunk=1, **bounds)
    assert (out == 0).all()


@pytest.mark.parametrize("new,old,h,g,d,rows", ALL_FORMS[:5])
@pytest.mark.parametrize("scale,k_exp,size", [(1e-38, 5, 1.0), (2.0 ** -140, 121, 1.0), (2.0 ** -140, 3, 2.0 ** 100), (3e38, 2, 2.0 ** -10), (3e38, 121, 0.0)])
def test_attention_scale_of_any_size(dev, new, old, h, g, d, rows, scale, k_exp, size):
    """Scales whose product with a block's leaves fp32's normal range, or whose own with log2 e does: softmax of what the scores are."""
    totals = [old + new - 13 * r for r in range(rows)]
    table, nb = random_table(totals, 0, seed=1)
    pages = random_pages(nb, g, d, seed=5)
    pages.k_exp.fill_(k_exp)
    q = (queries(rows * new, h, d, BF, seed=6).float() * size).to(BF)
    check_attention(q, pages, table, [new] * rows, totals, 1, scale=float(np.float32(scale)), max_new=new, max_kv=max(totals))

@pytest.mark.parametrize("new,old,h,g,d,rows", ALL_FORMS)
@pytest.mark.parametrize("size,dt", [(22, BF), (24, BF), (25, FP), (26, BF), (27, BF), (28, BF)])
def test_attention_near_ties_of_large_scores(dev, new, old, h, g, d, rows, size, dt):
    """Scores of 2^size and a little more, exact in fp32 (scale log2 e = 1): what counts is their difference, 0 to 24 in units of
    log2, so the bound has no part for the scores' own rounding (`top` = 24 for the exponential's argument)."""
    totals = [old + new - 13 * r for r in range(rows)]
    table, nb = random_table(totals, 0, seed=1)
    pages = random_pages(nb, g, d, seed=5)
    ulp = max(1, 2 ** (size - 23))
    gen = np.random.default_rng(size)
    pages.k.zero_()
    pages.k_exp.fill_(127)
    c = torch.full((nb, g, 32, 16), 0.0)
    c[..., :8] = 256
    diff = [x for x in (0, 8, 16, 24, ulp, 2 * ulp) if x % ulp == 0 and x <= 24 + ulp]
    c[..., 8] = torch.from_numpy(gen.choice(diff, (nb, g, 32)).astype(np.float32))
    for r, base in zip(range(rows), (0, ulp, 0, ulp, ulp, 0, 0)):
        c[int(table[r, 0]), :, :, 8] = base  # the reference is set here, by keys that later ones pass by 8 and more
    pages.k[:, :, 0] = c.to(torch.float8_e4m3fn).view(torch.uint8).cuda()
    q = torch.zeros(rows * new, h, d, device="cuda", dtype=dt)
    q[..., :8], q[..., 8] = 2.0 ** (size - 11), 1
    scale = float(np.float32(np.log(2)))
    assert np.float32(scale) * np.float32(1.4426950408889634) == 1
    k, v = scaled(pages)
    o, mag, _ = ok.attention(q.double().cpu().numpy(), k, v, table, starts([new] * rows), totals, scale, 1)
    out = kv8.attention(q, pages, torch.from_numpy(table).cuda(), ints(starts([new] * rows)), ints(totals), scale=scale, chunk=1, max_new=new, max_kv=max(totals))
    bound = attn_bound(o, mag, np.full(o.shape[:2], 24 + ulp), 1, dt)
    assert (np.abs(out.double().cpu().numpy() - o) <= bound).all()


@pytest.mark.parametrize("new,old,h,g,d,rows", ALL_FORMS[:5])
def test_attention_largest_score_takes_all(dev, new, old, h, g, d, rows):
    """Scores of 2^60 and more: the output is the winning key's value, which is exact in 16 bits.  (Scores whose first two lie
    within the fp32 rounding of D products, 2^-17 of their absolute sums, are left out: under 1% of them.)"""
    totals = [old + new - 13 * r for r in range(rows)]
    table, nb = random_table(totals, 0, seed=1)
    pages = random_pages(nb, g, d, seed=5)
    pages.k_exp.add_(60)
    q = queries(rows * new, h, d, BF, seed=6)
    k, v = scaled(pages)
    out = kv8.attention(q, pages, torch.from_numpy(table).cuda(), ints(starts([new] * rows)), ints(totals), scale=0.125, chunk=1, max_new=new,
                        max_kv=max(totals)).double().cpu().numpy()
    qd, left, n = q.double().cpu().numpy(), 0, 0
    for r, t in enumerate(totals):
        ids = table[r, :need(t)]
        for x in range(h):
            kk, vv = k[ids, x // (h // g)].reshape(-1, d)[:t], v[ids, x // (h // g)].reshape(-1, d)[:t]
            qq = qd[r * new:(r + 1) * new, x]
            s, a = qq @ kk.T, np.abs(qq) @ np.abs(kk).T
            hide = np.arange(t)[None] > t - new + np.arange(new)[:, None]
            s[hide], a[hide] = -np.inf, 0
            top = s.max(1, keepdims=True)
            sure = (s >= top - 2.0 ** -17 * a.max(1, keepdims=True)).sum(1) == 1
            assert np.array_equal(out[r * new:(r + 1) * new, x][sure], vv[s.argmax(1)][sure])
            none = hide.all(1)  # the first queries of a row with fewer keys than queries
            assert (out[r * new:(r + 1) * new, x][none] == 0).all()
            left, n = left + (~sure & ~none).sum(), n + (~none).sum()
    assert left <= 0.01 * n + 1


@pytest.mark.parametrize("new,old,h,g,d,rows", ALL_FORMS[1:3] + ALL_FORMS[4:])
def test_attention_queries_do_not_touch_each_other(dev, new, old, h, g, d, rows):
    """Queries of scores of 2^40 among the others, in the same tile and wave: the others' bits stay."""
    totals = [old + new] * rows
    table, nb = random_table(totals, 0, seed=1)
    pages = random_pages(nb, g, d, seed=5)
    q = queries(rows * new, h, d, BF, seed=6)
    hit = torch.zeros(rows * new, h, dtype=torch.bool, device="cuda")
    hit[1::9, 1::2] = True
    args = (pages, torch.from_numpy(table).cuda(), ints(starts([new] * rows)), ints(totals))
    kw = dict(scale=d ** -0.5, chunk=1, max_new=new, max_kv=max(totals))
    want = kv8.attention(q, *args, **kw)
    got = kv8.attention(torch.where(hit[..., None], q * 2.0 ** 40, q), *args, **kw)
    assert torch.isfinite(got).all() and torch.equal(got[~hit], want[~hit]) and not torch.equal(got[hit], want[hit])

@pytest.mark.parametrize("new,old,h,g,d,rows", ALL_FORMS[:5])
def test_attention_value_scale_byte_zero(dev, new, old, h, g, d, rows):
    """Values of scale 2^-127 (and a little more) are what they are, not zeros."""
    totals = [old + new - 13 * r for r in range(rows)]
    table, nb = random_table(totals, 0, seed=1)
    pages = random_pages(nb, g, d, seed=5)
    q = queries(rows * new, h, d, BF, seed=6)
    for low in (0, 2):
        pages.v_exp.copy_(torch.randint(0, low + 1, pages.v_exp.shape, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda"))
        out = check_attention(q, pages, table, [new] * rows, totals, 1, max_new=new, max_kv=max(totals))
        sees = torch.tensor([t - new + i >= 0 for t in totals for i in range(new)], device="cuda")  # rows of fewer keys than queries
        assert (out[sees].abs() > 0).double().mean() > 0.99 and (out[~sees] == 0).all()

def range_floor(q, pages, table, new, totals, scale, chunk):
    """Beside the relative rounding: a term's weight p_j 2^e_j is an fp16 number that may lie 2^10 below its query's reference
    before value scales are far apart, off by 2^-25 at most where the largest one is 2^(7 - 10) or more: 2^-22 of that a key."""
    k, _ = scaled(pages)
    size = np.broadcast_to(448.0 * np.exp2(pages.v_exp.cpu().numpy().astype(float) - 127)[..., None, None], k.shape)
    w, _, _ = ok.attention(q.double().cpu().numpy(), k, size, table, starts(new), totals, scale, chunk)
    return 2.0 ** -22 * max(totals) * w


def check_range(q, pages, table, new, totals, chunk, **kw):
    d = pages.head_dim
    k, v = scaled(pages)
    o, mag, top = ok.attention(q.double().cpu().numpy(), k, v, table, starts(new), totals, d ** -0.5, chunk)
    out = kv8.attention(q, pages, torch.from_numpy(table).cuda(), ints(starts(new)), ints(totals), scale=d ** -0.5, chunk=chunk, **kw)
    bound = attn_bound(o, mag, top, d, q.dtype) + range_floor(q, pages, table, new, totals, d ** -0.5, chunk)
    worst = float((np.abs(out.double().cpu().numpy() - o) / bound).max())
    assert worst <= 1, worst


@pytest.mark.parametrize("new,old,h,g,d,rows", ALL_FORMS)
@pytest.mark.parametrize("diff,below", [(24, 0), (24, 80), (40, 80), (40, 30), (60, 60), (100, 160), (120, 100)])
def test_attention_value_scales_far_apart(dev, new, old, h, g, d, rows, diff, below):
    """One block of values 2^diff times the others', its scores about 2^below times less likely: whichever of them counts is right.
    It stands first in some rows, in the middle or near the end in others."""
    totals = [old + new - 13 * r for r in range(rows)]
    table, nb = random_table(totals, 0, seed=1)
    pages = random_pages(nb, g, d, seed=5)
    pages.k_exp.fill_(121)
    pages.v_exp.fill_(100)
    q = queries(rows * new, h, d, BF, seed=6)
    w = 448 if below >= 80 else 256
    q[..., 0] = below * d ** 0.5 / (1.4427 * w * 2.0 ** -6)
    pages.k[:, :, 0, :, 0] = 0
    code = torch.tensor([-float(w)]).to(torch.float8_e4m3fn).view(torch.uint8).item()
    for r, t in enumerate(totals):
        b = int(table[r, (0, need(t) // 2, need(old) - 1)[(r + new) % 3]])
        pages.v_exp[b] = 100 + diff
        pages.k[b, :, 0, :, 0] = code if below else 0
    check_range(q, pages, table, [new] * rows, totals, 1, max_new=new, max_kv=max(totals))


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("new,old,h,g,d,rows", ALL_FORMS)
def test_attention_value_scales_of_every_size(dev, new, old, h, g, d, rows, dt):
    """Value scales drawn from 2^-60 to 2^8 for every block and head, in no order."""
    totals = [old + new - 13 * r for r in range(rows)]
    table, nb = random_table(totals, 0, seed=1)
    pages = random_pages(nb, g, d, seed=5)
    pages.v_exp.copy_(torch.randint(67, 132, pages.v_exp.shape, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda"))
    q = queries(rows * new, h, d, dt, seed=6)
    for size in (1, 12):
        check_range(q * size, pages, table, [new] * rows, totals, 1, max_new=new, max_kv=max(totals))


@pytest.mark.parametrize("new,old,h,g,d,rows", [(40, 100, 4, 2, 64, 3), (40, 100, 2, 2, 128, 3)] + ALL_FORMS[4:])
@pytest.mark.parametrize("last", [1, 2, 3])
def test_attention_unseen_scales_change_nothing(dev, new, old, h, g, d, rows, last):
    """The value scales of the row's last blocks 2^130 times the others': queries that see none of them keep their bits."""
    totals = [old + new] * rows
    table, nb = random_table(totals, 0, seed=1)
    pages = random_pages(nb, g, d, seed=5)
    q = queries(rows * new, h, d, BF, seed=6)
    args = (pages, torch.from_numpy(table).cuda(), ints(starts([new] * rows)), ints(totals))
    kw = dict(scale=d ** -0.5, chunk=1, max_new=new, max_kv=max(totals))
    want = kv8.attention(q, *args, **kw)
    first = (need(old + new) - last) * 32 - old  # the first query that sees one of them
    for r in range(rows):
        pages.v_exp[torch.from_numpy(table[r, need(old + new) - last:need(old + new)]).long().cuda()] = 250
    got = kv8.attention(q, *args, **kw)
    for r in range(rows):
        assert torch.equal(got[r * new:r * new + max(first, 0)], want[r * new:r * new + max(first, 0)])
        assert not torch.equal(got[r * new + max(first, 0):(r + 1) * new], want[r * new + max(first, 0):(r + 1) * new])

@pytest.mark.parametrize("new,old,h,g,d,rows", ALL_FORMS)
@pytest.mark.parametrize("keys", [True, False])
def test_attention_nan_scales(dev, new, old, h, g, d, rows, keys):
    """An E8M0 NaN among the keys' or the values' scales: NaN for every query that sees some of the block, the others as ever."""
    totals = [old + new] * rows
    table, nb = random_table(totals, 0, seed=1)
    pages = random_pages(nb, g, d, seed=5)
    q = queries(rows * new, h, d, BF, seed=6)
    args = (pages, torch.from_numpy(table).cuda(), ints(starts([new] * rows)), ints(totals))
    kw = dict(scale=d ** -0.5, chunk=1, max_new=new, max_kv=max(totals))
    want = kv8.attention(q, *args, **kw)
    b = need(old + new) - 1
    (pages.k_exp if keys else pages.v_exp)[int(table[0, b]), 1] = 255
    got = kv8.attention(q, *args, **kw)
    hit = torch.zeros(rows * new, h, dtype=torch.bool, device="cuda")
    hit[max(0, b * 32 - old):new, h // g:2 * (h // g)] = True
    assert got[hit].isnan().all() and torch.equal(got[~hit], want[~hit])
    k, v = pages.values([int(table[0, b])])
    assert (k if keys else v)[0, 1].isnan().all() and torch.isfinite((v if keys else k)[0]).all() and torch.isfinite(k[0, 0]).all()

def tile_parts_workspace():
    """What a call of the tile form in parts asks for (256 parts of 256 packed rows): no other form asks for as much."""
    return 256 * 256 * (128 + 2) * 4


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("G,g,rows,new,old", [(16, 8, 7, 32, 4100), (8, 8, 7, 63, 4100), (4, 8, 7, 127, 4100), (2, 8, 4, 250, 8200), (1, 32, 1, 250, 35000)])
def test_attention_tile_form_of_every_group(dev, dt, G, g, rows, new, old):
    """Groups of 16, 8, 4, 2 and 1 query heads in the tile form, its key lists in parts (the last one's of more than 128 blocks); the
    size of the workspace says that the form was taken."""
    import ctypes
    from t2w_amd import _lib
    totals = [old + new - 40 * r for r in range(rows)]
    table, nb = random_table(totals, 0, seed=G)
    pages = random_pages(nb, g, 128, seed=new)
    q = queries(rows * new, G * g, 128, dt, seed=g)
    a = _lib.KV8AttentionArgs(pages.struct, 1 << 20, 1 << 20, G * g * 128, G * g * 128, 0, rows * new, G * g, 1 << 20, table.shape[1], table.shape[1], 1 << 20,
                              1 << 20, rows, 1, 0.1, new, max(totals))
    assert _lib.lib().t2w_kv8_attention_workspace_bytes(ctypes.byref(a)) == tile_parts_workspace()
    check_attention(q, pages, table, [new] * rows, totals, 1, max_new=new, max_kv=max(totals))


@pytest.mark.parametrize("new,h,g,d", [(2, 4, 2, 64), (20, 4, 2, 128), (40, 2, 2, 128), (300, 2, 2, 128)])
def test_attention_rows_beyond_the_bound(dev, new, h, g, d):
    """A row of more new tokens than max_new says: NaN, or right; the others are right."""
    totals = [new + 100, 90, new + 7]
    table, nb = random_table(totals, 0, seed=1)
    pages = random_pages(nb, g, d, seed=5)
    q = queries(2 * new + 1, h, d, BF, seed=6)
    k, v = scaled(pages)
    new_l = [new, 1, new]
    o, mag, top = ok.attention(q.double().cpu().numpy(), k, v, table, starts(new_l), totals, d ** -0.5, 1)
    bound = attn_bound(o, mag, top, d, BF)
    for most in (1, max(1, new // 2), new - 1):
        out = kv8.attention(q, pages, torch.from_numpy(table).cuda(), ints(starts(new_l)), ints(totals), scale=d ** -0.5, chunk=1, max_new=most, max_kv=50)
        got = out.double().cpu().numpy()
        right = np.abs(got - o) <= bound
        for a, b in zip(starts(new_l), starts(new_l)[1:]):
            assert right[a:b].all() or (b - a > most and np.isnan(got[a:b]).all())


@pytest.mark.parametrize("h,g,d,rows,most,first", [(4, 2, 64, 75, 40, 1), (4, 2, 64, 75, 40, 70), (8, 1, 128, 20, 1, 7), (64, 32, 128, 10, 101, 3), (64, 32, 128, 75, 60, 60)])
@pytest.mark.parametrize("bounds", [False, True])
def test_attention_rows_of_a_larger_call(dev, h, g, d, rows, most, first, bounds):
    """The last rows of a call by slices of its tables; the tokens before them are left alone."""
    new = [(most, 1, 0, most // 2 + 1, most)[r % 5] for r in range(rows)]
    totals = [n + (0, 33, 70, 5)[r % 4] for r, n in enumerate(new)]
    table, nb = random_table(totals, 1, seed=rows)
    pages = random_pages(nb, g, d, seed=5)
    q = queries(sum(new), h, d, BF, seed=6)
    k, v = scaled(pages)
    o, mag, top = ok.attention(q.double().cpu().numpy(), k, v, table, starts(new), totals, d ** -0.5, 1)
    out = torch.full_like(q, 5)
    kw = {"max_new": most, "max_kv": max(totals)} if bounds else {}
    kv8.attention(q, pages, torch.from_numpy(table).cuda()[first:], ints(starts(new))[first:], ints(totals)[first:], scale=d ** -0.5, chunk=1, out=out, **kw)
    at = starts(new)[first]
    assert (out[:at] == 5).all()
    assert (np.abs(out.double().cpu().numpy() - o) <= attn_bound(o, mag, top, d, BF))[at:].all()

def test_graph_of_a_chunk_among_rows(dev):
    """One captured call in the tile form in parts serves other lengths: one row with all the tokens, some rows, every row, none;
    how many tiles there are, and so how many parts, is found at each replay."""
    rows, n_tok, h, g, d = 9, 256, 32, 8, 128
    table, nb = random_table([16900] * 2 + [300] * 7, 0, seed=1)
    pages = random_pages(nb, g, d, seed=2)
    q = queries(n_tok, h, d, BF, seed=3)
    dt, start, total = torch.from_numpy(table).cuda(), ints([0] * (rows + 1)), ints([0] * rows)
    out = torch.zeros_like(q)
    call = lambda: kv8.attention(q, pages, dt, start, total, scale=d ** -0.5, chunk=1, max_new=n_tok, max_kv=16900, out=out)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    k, v = scaled(pages)
    for new, kv in (([256] + [0] * 8, [16900, 5, 0, 0, 9, 0, 0, 0, 0]), ([100, 90, 0, 1, 30, 0, 20, 0, 15], [16900, 16000, 7, 300, 200, 0, 290, 0, 15]),
                    ([0] * 9, [0] * 9), ([28] * 9, [16900, 16900] + [300 - 30 * r for r in range(7)]), ([0, 200] + [0] * 7, [100, 16500] + [0] * 7)):
        start.copy_(ints(starts(new)))
        total.copy_(ints(kv))
        out.fill_(5)
        graph.replay()
        torch.cuda.synchronize()
        n = sum(new)
        o, mag, top = ok.attention(q.double().cpu().numpy(), k, v, table, starts(new), kv, d ** -0.5, 1)
        bound = attn_bound(o, mag, top, d, BF)
        assert (np.abs(out.double().cpu().numpy() - o) <= bound)[:n].all() and (out[n:] == 5).all()


# --- a run of them ----------------------------------------------------------------------------------------------------------

class Server:
    """A tiny server's loop over the three calls, and the same with the oracle."""

    def __init__(self, rows, h, g, d, dt, room, n_tok, seed=0):
        self.h, self.g, self.d, self.dt, self.rows = h, g, d, dt, rows
        self.nb = rows * room
        self.pages = random_pages(self.nb, g, d, seed=9)
        self.table = torch.full((rows, room), -1, dtype=torch.int32, device="cuda")
        self.free = torch.randperm(self.nb, generator=torch.Generator().manual_seed(seed)).int().cuda()
        self.kv, self.head = ints([0] * rows), ints([0])
        self.plan = kv8.KV8Plan(rows, n_tok)
        self.new = ints([0] * rows)
        self.x = torch.zeros(n_tok, h + 2 * g, d, device="cuda", dtype=dt)
        self.out = torch.zeros(n_tok, h, d, device="cuda", dtype=dt)

    def step(self, max_new, max_kv):
        """All on the GPU; the next step's lengths replace this one's at the end."""
        p, h, g = self.plan, self.h, self.g
        p.build(self.kv, self.new, self.table, self.free, self.head)
        kv8.append(self.pages, self.x[:, h:h + g], self.x[:, h + g:], self.table, p.row_start, p.kv_total, max_new=max_new)
        kv8.attention(self.x[:, :h], self.pages, self.table, p.row_start, p.kv_total, scale=self.d ** -0.5, chunk=1, max_new=max_new, max_kv=max_kv,
                      out=self.out)
        self.kv.copy_(p.kv_total)
        self.head.copy_(p.free_head)

    def check(self, state, new):
        """The step's results against the oracle, which goes on from its own state."""
        kc, vc, ke, ve, table, kv, head = state
        total, start, _, _, slots, head, status, table = ok.plan(kv, new, table, self.free.cpu().numpy(), head, self.plan.n_tok)
        assert status == 0 and int(self.plan.status) == 0
        assert self.plan.slots.tolist() == slots and np.array_equal(self.table.cpu().numpy(), table) and int(self.head) == head
        x = self.x.double().cpu().numpy()
        h, g = self.h, self.g
        ok.append(kc, vc, ke, ve, x[:, h:h + g], x[:, h + g:], table, start, total)
        for a, b in zip(host(self.pages), (kc, vc, ke, ve)):
            assert np.array_equal(a, b)
        o, mag, top = ok.attention(x[:, :h], kc * np.exp2(ke)[..., None, None], vc * np.exp2(ve)[..., None, None], table, start, total, self.d ** -0.5, 1)
        n = sum(new)
        got = self.out.double().cpu().numpy()[:n]
        assert (np.abs(got - o[:n]) <= attn_bound(o, mag, top, self.d, self.dt)[:n]).all()
        return kc, vc, ke, ve, table, total, head

    def state(self):
        return (*(x.astype(float) for x in host(self.pages)), self.table.cpu().numpy(), [0] * self.rows, 0)


@pytest.mark.parametrize("h,g,d,dt", [(4, 4, 64, BF), (8, 2, 128, FP)])
def test_prompts_then_steps(dev, h, g, d, dt):
    """Ragged prompts, then steps, some of rows that rest, then a second prompt chunk: every step against the oracle."""
    s = Server(3, h, g, d, dt, room=8, n_tok=160)
    state = s.state()
    gen = torch.Generator(device="cuda").manual_seed(1)
    for new in ([70, 33, 1], [1, 1, 1], [1, 0, 1], [0, 0, 0], [1, 1, 1], [2, 40, 31], [1, 1, 1]):
        s.x.copy_(torch.randn(s.x.shape, generator=gen, device="cuda"))
        s.new.copy_(ints(new))
        s.step(max(new), 256)
        torch.cuda.synchronize()
        state = s.check(state, new)


def test_graph_of_a_step(dev):
    """One captured graph serves steps of other lengths; between the replays the program works on and waits.  Every replay
    is checked against the oracle."""
    s = Server(3, 8, 2, 64, BF, room=6, n_tok=96)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s.step(0, 192)  # no new token: nothing changes
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.step(0, 192)
    state = s.state()
    gen = torch.Generator(device="cuda").manual_seed(2)
    for new in ([40, 3, 0], [1, 1, 1], [1, 1, 64], [0, 1, 1], [33, 1, 30]):
        s.x.copy_(torch.randn(s.x.shape, generator=gen, device="cuda"))
        s.new.copy_(ints(new))
        graph.replay()
        torch.cuda.synchronize()
        state = s.check(state, new)
        torch.randn(1 << 20, device="cuda").sum().item()


def test_two_graphs(dev):
    """Two captured graphs of long steps, replayed in turn and checked every time: their workspaces are their own."""
    totals = [5000, 4100]
    table, nb = random_table(totals, 0, seed=1)
    pages = random_pages(nb, 2, 128, seed=5)
    args = (pages, torch.from_numpy(table).cuda(), ints([0, 1, 2]), ints(totals))
    qs = [queries(2, 8, 128, BF, seed=s) for s in range(2)]
    want = [kv8.attention(q, *args, scale=0.1, max_new=1, max_kv=5000) for q in qs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(kv8.attention(q, *args, scale=0.1, max_new=1, max_kv=5000))
        graphs.append(g)
    for k in range(6):
        outs[k % 2].zero_()
        graphs[k % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[k % 2], want[k % 2])


def test_cache_error_against_16_bits(dev):
    """What the 8 bits cost: attention over the cache against attention over the keys and values themselves.  A code is off
    by at most 2^-4 of its value (and 2^-10 below e4m3's normal range, where the block's scale is at most 2^-8 of its
    largest value doubled), so with E = 2^-4 a score is off by at most E scale sum |q k| =: ds, a probability by a factor in
    exp(+-2 ds) and an output by E sum p |v| + (exp(2 ds) - 1) (1 + E) sum p |v|."""
    n, h, g, d = 200, 8, 2, 64
    s = Server(1, h, g, d, BF, room=8, n_tok=n)
    s.x.copy_(torch.randn(s.x.shape, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda"))
    s.new.copy_(ints([n]))
    s.step(n, 256)
    x = s.x.double().cpu()
    k, v = x[:, h:h + g].repeat_interleave(h // g, 1), x[:, h + g:].repeat_interleave(h // g, 1)
    p = torch.einsum("nhd,mhd->hnm", x[:, :h], k) * d ** -0.5
    p = torch.softmax(p.masked_fill(torch.ones(n, n).triu(1).bool(), -torch.inf), -1)
    ref = torch.einsum("hnm,mhd->nhd", p, v)
    err = (s.out.double().cpu() - ref).abs()
    low = 2.0 ** -10 * 2.0 ** -7  # a subnormal code's error, of the block's largest value
    E = 2.0 ** -4
    ak, av = k.abs() + low / E * k.abs().max(), v.abs() + low / E * v.abs().max()
    ds = E * torch.einsum("nhd,mhd->hnm", x[:, :h].abs(), ak).amax(-1).T[..., None] * d ** -0.5
    pv = torch.einsum("hnm,mhd->nhd", p, av)
    bound = E * pv + (torch.exp(2 * ds) - 1) * (1 + E) * pv + 2.0 ** -8 * ref.abs() + 2.0 ** -9 * pv
    assert (err <= bound).all()
