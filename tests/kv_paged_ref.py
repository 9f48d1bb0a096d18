"""Plain restatements of the paged cache's operators (include/kv_paged.h) in
Python lists and 64-bit numpy, for the tests."""
import numpy as np

NO_PAGES, NO_ROWS, BAD_LENGTH, BAD_PAGE, BAD_ROW = 1, 2, 4, 8, 16


def pages_of(tokens, page):
    return -(-tokens // page)


def map_step(length, start, end, table, free, page, n_pages, max_rows):
    """One kv_paged_map call on lists: (error bits, table, free stack, rows
    [(request, position, slot)], row0). table and free are not changed."""
    n, blocks = len(length), len(table[0])
    zeros = [0] * (n + 1)
    for a, s, e in zip(length, start, end):
        if s < 0 or s > a or e < s or e > blocks * page or a > blocks * page:
            return BAD_LENGTH, table, free, [], zeros
    table = [list(t) for t in table]
    stack = list(free)
    for i in range(n):
        stack += table[i][pages_of(end[i], page):pages_of(length[i], page)]
    need = sum(max(0, pages_of(e, page) - pages_of(a, page)) for a, e in zip(length, end))
    rows_n = sum(e - s for s, e in zip(start, end))
    code = (NO_ROWS if rows_n > max_rows else 0) | (NO_PAGES if need > len(stack) else 0)
    if code == 0 and len(stack) - need > n_pages:
        code = BAD_LENGTH
    if code:
        return code, [list(t) for t in table], free, [], zeros
    rows, row0 = [], [0]
    for i in range(n):
        for b in range(pages_of(length[i], page), pages_of(end[i], page)):
            table[i][b] = stack.pop()
        for p in range(start[i], end[i]):
            pg = table[i][p // page]
            if 0 <= pg < n_pages:
                rows.append((i, p, pg * page + p % page))
            else:
                rows.append((i, p, -1))
                code |= BAD_PAGE
        row0.append(len(rows))
    return code, table, stack, rows, row0


def turn(x, rope, pos, dim, dtype):
    """x [rows][heads][hs] turned in `dtype`, one rounding per product and sum."""
    x = x.astype(dtype).copy()
    c = rope[pos][:, None, 0:dim:2].astype(dtype)
    s = rope[pos][:, None, 1:dim:2].astype(dtype)
    a, b = x[..., 0:dim:2].copy(), x[..., 1:dim:2].copy()
    x[..., 0:dim:2] = a * c - b * s
    x[..., 1:dim:2] = a * s + b * c
    return x


def rope_table(length, dim, base=10000.0):
    i = np.arange(dim // 2)
    ang = np.arange(length)[:, None] * base ** (-2.0 * i / max(dim, 1))[None]
    return np.stack([np.cos(ang), np.sin(ang)], 2).reshape(length, dim).astype(np.float32)


def attend(q, keys, values, scale):
    """One row: q [heads][hs], keys and values [tokens][kv_heads][hs] -> (out,
    weight) in 64 bits; weight [heads][hs] is sum_t p_t |v_t|, and the third
    is max_t sum_d |scale q_d k_td| per head."""
    h, hs = q.shape
    t, kvh, _ = keys.shape
    if t == 0:
        return np.zeros((h, hs)), np.zeros((h, hs)), np.zeros(h)
    k = np.repeat(keys.astype(np.float64), h // kvh, axis=1)
    v = np.repeat(values.astype(np.float64), h // kvh, axis=1)
    q = q.astype(np.float64)
    s = scale * np.einsum("hd,thd->ht", q, k)
    e = np.exp(s - s.max(1, keepdims=True))
    p = e / e.sum(1, keepdims=True)
    size = abs(scale) * np.einsum("hd,thd->ht", np.abs(q), np.abs(k)).max(1)
    return np.einsum("ht,thd->hd", p, v), np.einsum("ht,thd->hd", p, np.abs(v)), size


def attend_tolerance(weight, size, hs, tokens):
    """How far a 32-bit attention may be off, per output: a score of hs
    products is off by at most (hs + 8) 2^-24 of its products' sizes (8: the
    operands' splitting into two parts of 11 bits, 2^-22 each side, and the
    scale), its exponential by twice that plus 2^-21 (the score's own
    rounding in base 2 and the exponential's error, both relative to a
    score of up to 2^2 size), the sums of `tokens` terms above and below by
    tokens 2^-24 each, the division by 2^-23."""
    ds = (hs + 8) * 2.0 ** -24 * size[:, None]
    return weight * (2 * ds + 2.0 ** -21 * (1 + size[:, None]) + 2 * tokens * 2.0 ** -24 + 2.0 ** -23) + 1e-30
