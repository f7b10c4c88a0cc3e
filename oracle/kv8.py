"""The paged 8-bit key/value cache in plain float64: tables from request lengths, the quantizing append, attention.

No counterpart in the reference (its key/value pools are 16-bit, ``engine/runtime/dit_fast.py:59-64``): this restates the
operators' own definition (``include/t2w.h``, t2w_kv8_*), with loops over rows, blocks and heads.
"""

from __future__ import annotations

import numpy as np

BLOCK = 32


def e4m3(x: np.ndarray) -> np.ndarray:
    """x rounded to the nearest OCP e4m3 value, ties to even (quantum 2^-9 at the bottom; |x| <= 448 is the caller's)."""
    a = np.abs(x)
    e = np.floor(np.log2(np.where(a > 0, a, 1.0)))
    q = np.exp2(np.maximum(e, -6.0) - 3.0)
    return np.rint(x / q) * q


def exponent(amax: float) -> int:
    """The smallest e with amax <= 448 * 2^e, in [-126, 126] (-126 below fp32's normal range)."""
    if amax < 2.0 ** -126:
        return -126
    e = int(np.floor(np.log2(amax))) - 8
    e += amax > 448.0 * 2.0 ** e
    return min(126, max(-126, e))


def plan(kv_len, new_len, table, free_ids, free_head, n_tok):
    """Returns (kv_total, row_start, tok_row, tok_pos, slots, free_head, status, table) as int lists / arrays."""
    R, width = len(kv_len), table.shape[1]
    need = lambda n: -(-n // BLOCK)  # noqa: E731
    status = 0
    if any(x < 0 for x in list(kv_len) + list(new_len)):
        status |= 1
    if sum(new_len) > n_tok:
        status |= 2
    if any(need(k + n) > width for k, n in zip(kv_len, new_len)):
        status |= 4
    more = [need(k + n) - need(k) for k, n in zip(kv_len, new_len)]
    if free_head < 0 or free_head + sum(more) > len(free_ids):
        status |= 8
    blank = [-1] * n_tok
    if status:
        return list(kv_len), [0] * (R + 1), blank, blank, blank, free_head, status, table
    table = table.copy()
    start, rows, pos, slots = [0], [], [], []
    for r in range(R):
        for b in range(need(kv_len[r]), need(kv_len[r] + new_len[r])):
            table[r, b] = free_ids[free_head]
            free_head += 1
        for p in range(kv_len[r], kv_len[r] + new_len[r]):
            rows.append(r)
            pos.append(p)
            slots.append(int(table[r, p // BLOCK]) * BLOCK + p % BLOCK)
        start.append(start[-1] + new_len[r])
    pad = blank[len(rows):]
    return [k + n for k, n in zip(kv_len, new_len)], start, rows + pad, pos + pad, slots + pad, free_head, 0, table


def append(kc, vc, ke, ve, k, v, table, row_start, kv_total):
    """In place: code values kc, vc float64 [blocks, heads, 32, D] (NaN for the NaN code), exponents ke, ve int
    [blocks, heads]; k, v [n_tok, heads, D]."""
    for r in range(len(kv_total)):
        old = kv_total[r] - (row_start[r + 1] - row_start[r])
        p = old
        while p < kv_total[r]:
            b, first = int(table[r, p // BLOCK]), p % BLOCK
            n = min(BLOCK - first, kv_total[r] - p)
            t0 = row_start[r] + p - old
            p += n
            if not 0 <= b < kc.shape[0]:
                continue
            for h in range(kc.shape[1]):
                kk, vv = k[t0:t0 + n, h].astype(np.float64), v[t0:t0 + n, h].astype(np.float64)
                bad = ~(np.isfinite(kk).all(1) & np.isfinite(vv).all(1))
                for x, c, e, key in ((kk, kc, ke, True), (vv, vc, ve, False)):
                    x = np.where(bad[:, None], 0.0, x)
                    new = exponent(float(np.abs(x).max()))
                    if first == 0:
                        c[b, h] = 0.0
                        e[b, h] = new
                    elif new > e[b, h]:
                        c[b, h, :first] = e4m3(c[b, h, :first] * 2.0 ** float(e[b, h] - new))
                        e[b, h] = new
                    c[b, h, first:first + n] = e4m3(x * 2.0 ** -float(e[b, h]))
                    if key:
                        c[b, h, first:first + n][bad] = np.nan


def attention(q, keys, vals, table, row_start, kv_total, scale, chunk):
    """q [n_tok, heads, D] float64; keys, vals [blocks, kv_heads, 32, D] float64.  Returns the outputs, the sums
    sum_j p_j |v_j| and the largest scale * sum_d |q_d k_d| of each (token, head): what the error bounds are made of."""
    N, H, D = q.shape
    G = keys.shape[1]
    out, mag, top = np.zeros((N, H, D)), np.zeros((N, H, D)), np.zeros((N, H))
    for r in range(len(kv_total)):
        a, b, total = row_start[r], row_start[r + 1], kv_total[r]
        i = np.arange(b - a)
        see = total - (b - a) + (b - a if chunk == 0 else np.minimum(b - a, (i // chunk + 1) * chunk)) + 0 * i
        if b == a or see.max() <= 0:
            continue
        ids = table[r, :-(-total // BLOCK)]
        hide = np.arange(total)[None] >= see[:, None]
        for h in range(H):
            g = h // (H // G)
            kk, vv = keys[ids, g].reshape(-1, D)[:total], vals[ids, g].reshape(-1, D)[:total]
            s = np.where(hide, -np.inf, q[a:b, h] @ kk.T * scale)
            m = s.max(1, keepdims=True)
            p = np.exp(s - np.where(np.isfinite(m), m, 0.0))
            p /= np.maximum(p.sum(1, keepdims=True), 1e-300)
            out[a:b, h], mag[a:b, h] = p @ vv, p @ np.abs(vv)
            top[a:b, h] = scale * np.where(hide, 0.0, np.abs(q[a:b, h]) @ np.abs(kk).T).max(1)
    return out, mag, top
