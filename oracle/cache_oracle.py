"""Oracle of the 8-bit paged cache in float64 and plain loops: block tables, append, attention over the cache (test infrastructure only)."""
import numpy as np

TOP, MIN_EXP = 448.0, -118


def e4m3_values():
    """The value of every e4m3 code (NaN for 0x7f and 0xff)."""
    out = np.zeros(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = (m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        out[c] = np.nan if c & 127 == 127 else -x if c & 128 else x
    return out


VALUES = e4m3_values()


def to_code(x):
    """Nearest e4m3 code of float64 numbers up to 448 in magnitude, ties to the even code; the NaN code for what is not finite."""
    grid = VALUES[:127]  # codes of ascending magnitudes; the parity of a code is that of its mantissa
    a = np.abs(np.where(np.isfinite(x), x, 0.0))
    hi = np.clip(np.searchsorted(grid, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up, down = grid[hi] - a, a - grid[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = np.where(grid[hi] == a, hi, code)
    return np.where(np.isfinite(x), code | np.where(np.signbit(x), 128, 0), 127).astype(np.uint8)


def scale_for(a):
    e = MIN_EXP
    while a > TOP * 2.0 ** e:
        e += 1
    return 2.0 ** e


def pieces_bound(requests, tokens, page):
    m = min(requests, tokens)
    return m + min(m, tokens - m) + max(0, tokens - 2 * m) // page


def blocks(lengths, new, tables, free, count, page, tokens):
    """(lengths, count, ends, slots, pieces, tables, free) after the step, or None where it is refused."""
    R, width = tables.shape
    tables, free = tables.copy(), free.copy()
    up = lambda x: -(-x // page)  # noqa: E731
    after = [int(t) + int(n) for t, n in zip(lengths, new)]
    if any(not 0 <= t <= width * page for t in list(lengths) + after) or sum(max(0, int(n)) for n in new) > tokens:
        return None
    stack = [int(x) for x in free[:count]]
    for r in range(R):
        stack += [int(x) for x in tables[r, up(after[r]):up(int(lengths[r]))]]
    if sum(max(0, up(a) - up(int(t))) for a, t in zip(after, lengths)) > len(stack):
        return None
    for r in range(R):
        for b in range(up(int(lengths[r])), up(after[r])):
            tables[r, b] = stack.pop()
    free[count:len(stack)] = stack[count:]
    slots, pieces = np.full(tokens, -1), []
    ends, row = [], 0
    for r in range(R):
        t, n = int(lengths[r]), max(0, int(new[r]))
        for i in range(n):
            slots[row + i] = tables[r, (t + i) // page] * page + (t + i) % page
        for b in range(t // page, up(t + n)) if n else ():
            old, stop = max(0, t - b * page), min(page, t + n - b * page)
            pieces.append((tables[r, b], row + max(0, b * page - t), old, stop - old))
        row += n
        ends.append(row)
    pieces += [(-1, 0, 0, 0)] * (pieces_bound(R, tokens, page) - len(pieces))
    return np.array(after), len(stack), np.array(ends), slots, np.array(pieces).reshape(-1, 4), tables, free


def append(x, codes, scales, pieces):
    """x [heads, tokens, dim] float64 into copies of codes (uint8 [pages, heads, page, row]) and scales (float64)."""
    codes, scales = codes.copy(), scales.astype(np.float64)
    dim = x.shape[-1]
    for page, first, old, n in pieces:
        if page < 0:
            continue
        for h in range(x.shape[0]):
            part = x[h, first:first + n]
            fin = np.abs(part[np.isfinite(part)])
            s = scale_for(fin.max() if fin.size else 0.0)
            if old:
                if scales[page, h] >= s:
                    s = scales[page, h]
                else:
                    c = codes[page, h, :old]
                    codes[page, h, :old] = np.where(c & 127 == 127, c, to_code(VALUES[c] * (scales[page, h] / s)))
            codes[page, h, old:old + n, :dim] = to_code(part / s)
            codes[page, h, old:old + n, dim:] = 0
            scales[page, h] = s
    return codes, scales


def attend(q, k, v, n, inv_temp, attend_current, own_v=None, wide=False):
    """One request and head in float64: q [n, D] are the last n of the L tokens of k, v [L, D].  Returns (o, rem) and, for each, a bound on
    what float32 arithmetic may be off: products summed in any order with truncated accumulations, 2 (D + 4) 2^-24 of the sum of magnitudes, which the
    weights feel once through their own score and sum(beta) times through the others; 64 steps of 2^-24 for exponentials, logarithms
    and the two-term weights; sums of logarithms over blocks of 32 keys.  ``wide``: the kernel for many queries, which rounds its weights to that many bfloat16 terms (2^-8 each), multiplies 1 - beta
in float32 (four roundings of 2^-23 a key) and lets no 1 - beta fall below 2^-30."""
    L, D = k.shape
    u = 2.0 ** -24
    o, rem, to, tr = np.zeros((n, D)), np.ones(n), np.zeros((n, D)), np.zeros(n)
    for i in range(n):
        m = L - n + i + (1 if attend_current else 0)
        if m > 0:
            x = (k[:m] @ q[i]) * inv_temp
            ex = 2 * (D + 4) * u * (np.abs(k[:m]) @ np.abs(q[i])).max() * abs(inv_temp)
            soft = np.maximum(x, 0) + np.log1p(np.exp(-np.abs(x)))
            right = np.cumsum(soft[::-1])[::-1] - soft
            beta = 1 / (1 + np.exp(-x))
            a = beta * np.exp(-right)
            o[i], rem[i] = a @ v[:m], np.exp(-soft.sum())
            with np.errstate(invalid="ignore", over="ignore"):
                off = np.minimum(1.0, np.expm1(ex * (1 + beta.sum()) + u * (64 + (m / 32 + 8) * right)) + (2.0 ** (-8 * wide) * 1.01 + 8 * m * u if wide else 0))
                to[i] = (a * off) @ np.abs(v[:m]) + 2 * (m / 32 + 40) * u * (a @ np.abs(v[:m]))
                tr[i] = rem[i] * min(1.0, np.expm1(ex * beta.sum() + u * (64 + (m / 32 + 8) * soft.sum())) + (8 * m * u if wide else 0))
                if wide:
                    to[i] += 2.0 ** -29 * np.abs(v[:m]).max(0)
                    tr[i] += 2.0 ** -29
        if own_v is not None:
            o[i] += rem[i] * own_v[i]
            to[i] += tr[i] * np.abs(own_v[i])
    return o, rem, to, tr


def attend_rows(q, k, v, n, inv_temp, attend_current, own_v=None, wide=0):
    """attend(), all rows at once: for tests with many of them."""
    (L, D), u, m = k.shape, 2.0 ** -24, (k.shape[0] - n + np.arange(n) + (1 if attend_current else 0))[:, None]
    if L == 0 or n == 0:
        return np.zeros((n, D)), np.ones(n), np.zeros((n, D)), np.zeros(n)
    sees = np.arange(L)[None] < m
    x = np.where(sees, (q @ k.T) * inv_temp, 0.0)
    ex = 2 * (D + 4) * u * np.where(sees, np.abs(q) @ np.abs(k).T, 0.0).max(1, keepdims=True) * abs(inv_temp)
    soft = np.where(sees, np.maximum(x, 0) + np.log1p(np.exp(-np.abs(x))), 0.0)
    total = soft.sum(1, keepdims=True)
    right = np.cumsum(soft[:, ::-1], 1)[:, ::-1] - soft
    beta = np.where(sees, 1 / (1 + np.exp(-x)), 0.0)
    mass = beta.sum(1, keepdims=True)
    a, rem, some = beta * np.exp(-right), np.exp(-total), m > 0
    with np.errstate(invalid="ignore", over="ignore"):
        off = np.minimum(1.0, np.expm1(ex * (1 + mass) + u * (64 + (m / 32 + 8) * right)) + (2.0 ** (-8 * wide) * 1.01 + 8 * m * u if wide else 0))
        tr = np.where(some, rem * np.minimum(1.0, np.expm1(ex * mass + u * (64 + (m / 32 + 8) * total)) + (8 * m * u if wide else 0)), 0.0)
    to = (a * off) @ np.abs(v) + 2 * (m / 32 + 40) * u * (a @ np.abs(v))
    if wide:
        top = np.maximum.accumulate(np.abs(v), 0)[np.maximum(m[:, 0], 1) - 1]
        to, tr = to + np.where(some, 2.0 ** -29 * top, 0.0), tr + np.where(some, 2.0 ** -29, 0.0)
    o, rem, tr = a @ v, rem[:, 0], tr[:, 0]
    if own_v is not None:
        o, to = o + rem[:, None] * own_v, to + tr[:, None] * np.abs(own_v)
    return o, rem, to, tr


def tiles_of_blocks(lengths, new, kv, shared, blocks, attend_current=False, tile=256, step=128, cost=2):
    """How the kernel for many queries deals its tiles to `blocks` blocks: per block, in order, (columns, steps that the block does) of every tile."""
    see = 1 if attend_current else 0
    jobs = []  # (columns, steps, steps of keys that the tile does not see)
    for length, n in zip(lengths, new):
        steps = max(1, -(-(length - 1 + see) // step))
        for _ in range(kv):
            for c0 in range(0, n * shared, tile):
                cols = min(tile, n * shared - c0)
                keys = length - n + (c0 + cols - 1) // shared + see
                jobs.append((cols, steps, steps - max(1, -(-keys // step))))
    units = sum(s + cost for _, s, _ in jobs)
    shares = max(1, min(blocks, units))
    out, at = [[] for _ in range(shares)], 0
    for cols, steps, unseen in jobs:
        first, last = at, at + steps + cost
        at = last
        for b in range(first * shares // units, shares):
            lo, hi = max(first, units * b // shares), min(last, units * (b + 1) // shares)
            if lo >= last:
                break
            if lo < hi:
                out[b].append((cols, max(0, max(0, hi - first - cost) - max(max(0, lo - first - cost), unseen))))
    return out
