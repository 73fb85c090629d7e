"""Plain 64-bit restatement of the 4-bit key/value cache (include/zvdb_hip.h: "4-bit key/value cache") for the tests: numpy, loops, no library code."""
import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)


def width(d):
    return 64 if d <= 64 else 128 if d <= 128 else 256


def head_bytes(d, page):
    return page * (width(d) + width(d) // 16)


def encode_rows(x, d):
    """(codes [n, D], scale bytes [n, D/32], values [n, d] in fp64; NaN where the block is) of rows x [n, d], exact fp32 or bf16 numbers."""
    w = width(d)
    rows = np.zeros((len(x), w))
    rows[:, :d] = x
    blocks = rows.reshape(len(x), w // 32, 32)
    fine = np.isfinite(blocks).all(-1)
    clean = np.where(fine[..., None], blocks, 0.0)
    top = np.abs(clean).max(-1)
    m, e = np.frexp(top)  # top = m 2^e, 1/2 <= m < 1
    e = np.where(top == 0, -125, np.clip(e - 1 + (m >= 0.875) - 2, -125, 125))
    y = np.abs(clean) / np.exp2(e.astype(np.float64))[..., None]
    far = np.abs(y[..., None] - GRID)
    best = far == far.min(-1, keepdims=True)
    tie = best.sum(-1) > 1  # two neighbours: the even one of them
    even = best & (np.arange(8) % 2 == 0)
    codes = np.where(tie, even.argmax(-1), best.argmax(-1)).astype(np.uint8)
    codes = np.where(fine[..., None], codes | np.where(np.signbit(blocks), 8, 0).astype(np.uint8), 0).astype(np.uint8)
    vals = GRID[codes & 7] * np.where(codes & 8, -1.0, 1.0) * np.exp2(e.astype(np.float64))[..., None]
    vals = np.where(fine[..., None], vals, np.nan).reshape(len(x), w)[:, :d]
    return codes.reshape(len(x), w), np.where(fine, e + 127, 255).astype(np.uint8), vals


def put(cache, d, heads, page, slot, head, codes, scales, value):
    """Writes one row's codes and scales into the bytes of a cache [pages * page bytes]."""
    w = width(d)
    nb = w // 32
    hb = head_bytes(d, page)
    base = (slot // page) * heads * hb + head * hb
    t = slot % page
    half = page * w // 2
    for e in range(w):
        if not value:
            at = base + t * (w // 2) + e // 2
        else:
            piece, within = e // (2 * nb), e % (2 * nb)
            at = base + half + (t // 4) * 64 * nb + piece * 4 * nb + (t % 4) * nb + within // 2
        if e % 2 == 0:
            cache[at] = (cache[at] & 0xF0) | codes[e]
        else:
            cache[at] = (cache[at] & 0x0F) | (codes[e] << 4)
    for b in range(nb):
        at = base + 2 * half + (t * nb + b if not value else page * nb + (t // 4) * 4 * nb + b * 4 + t % 4)
        cache[at] = scales[b]


def plan(lengths, new, ring, cursor, tables, page, pages, slot_cap):
    """(status code, starts, slots, out lengths, out cursor, tables, pages needed, tokens), token by token."""
    n, stride = len(lengths), tables.shape[1]
    lengths, new = [int(x) for x in lengths], [int(x) for x in new]
    need = [-(-(c + a) // page) - -(-c // page) for c, a in zip(lengths, new)]
    total, pages_needed = sum(new), sum(need)
    empty = np.full(slot_cap, -1, np.int64)
    left = min(max(int(cursor[1]) - int(cursor[0]), 0), len(ring))
    code = 0
    if any(-(-(c + a) // page) > stride or c + a > 2 ** 31 - 1 for c, a in zip(lengths, new)):
        code = 2
    elif total > slot_cap:
        code = 3
    elif pages_needed > left:
        code = 1
    if code:
        return code, np.zeros(n + 1, np.int64), empty, lengths, list(cursor), tables.copy(), pages_needed, total
    tables, slots, starts, taken = tables.copy(), empty, [0], int(cursor[0])
    at = 0
    for i in range(n):
        for pos in range(lengths[i], lengths[i] + new[i]):
            if pos % page == 0:
                tables[i, pos // page] = ring[taken % len(ring)]
                taken += 1
            p = int(tables[i, pos // page])
            slots[at] = p * page + pos % page if 0 <= p < pages else -1
            at += 1
        starts.append(at)
    return 0, np.array(starts), slots, [c + a for c, a in zip(lengths, new)], [taken, int(cursor[1])], tables, pages_needed, total


def attend_row(q, k, v, scale, kind):
    """(o, lse, bound of o per element, bound of lse) of one row over the tokens k, v [t, d] that it sees, in 64 bits.

    Bounds.  u = 2^-24 (half a step of fp32).  Scores: the matrix instruction adds d products (three times as many with fp32 queries:
    24-bit terms) with at most a step, 2 u, lost for each, scaled by a constant that is off by 2 u and subtracted from the maximum with one
    rounding of a number up to twice the largest score: ds = 2 u (3 d + 3) scale sum|q k| + 4 u (max|s| + 8 ln 2).  exp2 is off by 2 u
    (one step) of itself, so a weight is off by dw = ds + 4 u of itself, numerator and denominator both.  Sums over t tokens, the joins of at
    most 4 waves and 256 splits and their factors: (t + 600) 2 u.  bf16: P is off by half a step, 2^-8, in the numerator; the output by 2^-8 of
    itself.  fp32: P's three terms leave 2^-24 of it, the output is off by u."""
    t, d = k.shape
    u = 2.0 ** -24
    if t == 0:
        return np.zeros(d), -np.inf, np.zeros(d), 0.0
    s = scale * (k @ q)
    top = s.max()
    p = np.exp(s - top)
    l = p.sum()
    o, lse = (p @ v) / l, top + np.log(l)
    mass = (p @ np.abs(v)) / l
    ds = 2 * u * (3 * d + 3) * np.max(scale * (np.abs(k) @ np.abs(q))) + 4 * u * (np.max(np.abs(s)) + 8 * np.log(2))
    sums = (t + 600) * 2 * u
    half = 2.0 ** -8 if kind == "bf16" else u
    bound = mass * (2 * (ds + 4 * u) + 2 * sums + half) * 1.01 + half * np.abs(o) * 1.01 + 1e-37
    return o, lse, bound, (ds + 4 * u + sums + 4 * u * abs(lse)) * 1.01 + 2 * u
