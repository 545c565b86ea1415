"""The paged cache's operators (superslm_amd/cache_ops.py) and sampling on the host, one token, page or row after the
other in Python's integers and the oracle's primitives: what the GPU tests compare against, bit for bit."""
import numpy as np

import batch_ops_ref as ref

MAX_SHIFT, MAX_UNITS = 8, 127 << 8
POSITION, MANTISSA = 9, 4
INVALID, EXHAUSTED = 1, 14


def round_away(x, e):
    """x / 2^e to the nearest, ties away from zero; arrays or integers."""
    half = (1 << e) >> 1
    return np.sign(x) * ((np.abs(x) + half) >> e)


class Layout:
    """A layer's place in a page of `p` positions: `lead` bytes before it, `tail` behind it."""

    def __init__(self, kv_heads, dim, p, lead=0, tail=0):
        self.nkv, self.d, self.p = kv_heads, dim, p
        self.half = kv_heads * p * dim
        self.k_offset, self.v_offset = lead, lead + self.half
        self.exp_offset = lead + 2 * self.half
        self.page_bytes = (self.exp_offset + 2 * kv_heads + tail + 15) // 16 * 16

    def codes(self, pool, page, i):
        """K (i = 0) or V codes of a page, a view [kv_heads, p, d]."""
        at = (self.k_offset, self.v_offset)[i]
        return pool[page, at:at + self.half].reshape(self.nkv, self.p, self.d)

    def exps(self, pool, page, i):
        at = self.exp_offset + i * self.nkv
        return pool[page, at:at + self.nkv].view(np.uint8)

    def values(self, pool, table, width):
        """K and V in units, [kv_heads, width, d] each."""
        out = [np.zeros((self.nkv, width, self.d), np.int64) for _ in range(2)]
        for i in range(2):
            for n in range(-(-width // self.p)):
                m = min(self.p, width - n * self.p)
                e = np.minimum(self.exps(pool, table[n], i), MAX_SHIFT).astype(np.int64)
                out[i][:, n * self.p:n * self.p + m] = self.codes(pool, table[n], i)[:, :m].astype(np.int64) << e[:, None, None]
        return out


def land(code, m, e, r_t, e_t):
    """The reference's landing of one code: round_away(code m r_t / 2^k), unclamped."""
    k = max(-4096, min(4096, 62 - (e - e_t)))
    x = abs(code * m) * r_t
    y = (2 * x + (1 << k)) >> (k + 1) if k >= 0 else x << -k
    return -y if (code < 0) != (m < 0) else y


def rotate(x, cos, sin, halves):
    """One head's values: the first 2 len(cos) of them turn."""
    y, n = x.copy(), len(cos)
    for i in range(n):
        a, b = (i, i + n) if halves else (2 * i, 2 * i + 1)
        y[a] = round_away(int(x[a]) * int(cos[i]) - int(x[b]) * int(sin[i]), 30)
        y[b] = round_away(int(x[a]) * int(sin[i]) + int(x[b]) * int(cos[i]), 30)
    return y


def need(x):
    """The least exponent that keeps the codes of these values within 127."""
    e = 0
    while int(round_away(int(np.abs(x).max()), e)) > 127:
        e += 1
    return e


def store_token(lay, pool, table, pos, q, k, v, k_scale, v_scale, units, cos, sin, halves):
    """One token of one row: q [heads, d], k and v [kv_heads, d] codes.  (rotated q, values clamped)."""
    clamped, out = 0, np.zeros_like(q)
    for h in range(q.shape[0]):
        out[h] = np.clip(rotate(q[h].astype(np.int64), cos, sin, halves), -127, 127)
    page, slot = table[pos // lay.p], pos % lay.p
    for i, (x, (m, e)) in enumerate(((k, k_scale), (v, v_scale))):
        for j in range(lay.nkv):
            r_t, e_t = units[i][j]
            y = [land(int(c), int(m), int(e), r_t, e_t) for c in x[j]]
            clamped += sum(abs(c) > MAX_UNITS for c in y)
            y = np.array([max(-MAX_UNITS, min(MAX_UNITS, c)) for c in y], np.int64)
            if i == 0:
                y = rotate(y, cos, sin, halves)
                clamped += int((np.abs(y) > MAX_UNITS).sum())
                y = np.clip(y, -MAX_UNITS, MAX_UNITS)
            codes, exps = lay.codes(pool, page, i), lay.exps(pool, page, i)
            was = 0 if slot == 0 else min(int(exps[j]), MAX_SHIFT)
            now = max(was, need(y))
            if now > was:
                codes[j, :slot] = round_away(codes[j, :slot].astype(np.int64), now - was)
            exps[j] = now
            codes[j, slot] = round_away(y, now)
    return out, clamped


def attention_token(lib, q, q_scale, khead, k, v, fold):
    """k, v [kv_heads, width, d] in units."""
    return ref.attention_row(lib, q, q_scale, khead, k, v, fold)


def update(tables, lengths, source, keep, room, p, pages, held=None):
    """(result, new tables, pages to copy as [(from, to)]); tables None when the call changes nothing."""
    rows, width = tables.shape
    for r in range(rows):
        s, n = int(source[r]), 0
        ok = -1 <= s < rows
        if ok and s >= 0:
            n = int(lengths[s])
        ok = ok and 0 <= n <= width * p and 0 <= keep[r] <= n and keep[r] <= room[r] <= width * p
        if ok and s >= 0:
            t = tables[s, :-(-int(keep[r]) // p)]
            ok = bool(((t >= 0) & (t < pages)).all())
        if not ok:
            return [INVALID, 0, 0, r], None, []
    kept = [tables[source[r], :-(-int(keep[r]) // p)].tolist() if source[r] >= 0 else [] for r in range(rows)]
    writes = [keep[r] % p != 0 and room[r] > keep[r] for r in range(rows)]
    holders = {}
    for r, t in enumerate(kept):
        for i, x in enumerate(t):
            holders.setdefault(x, []).append((r, bool(writes[r]) and i == len(t) - 1))
    free = [x for x in range(pages) if x not in holders and not (held is not None and held[x])]
    out, used, copies = np.full_like(tables, -1), 0, []
    for r, t in enumerate(kept):
        t = list(t)
        if writes[r]:
            x = t[-1]
            other = list(holders[x])
            other.remove((r, True))
            if (held is not None and held[x]) or any(not w or o < r for o, w in other):
                copies.append((x, used))
                t[-1] = ~used
                used += 1
        while len(t) < -(-int(room[r]) // p):
            t.append(~used)
            used += 1
        kept[r] = t
    if used > len(free):
        return [EXHAUSTED, len(free) - used, 0, -1], None, []
    for r, t in enumerate(kept):
        out[r, :len(t)] = [x if x >= 0 else free[~x] for x in t]
    return [0, len(free) - used, len(copies), -1], out, [(a, free[b]) for a, b in copies]


def compact(tables, lengths, p, pages, held=None):
    """(result, new tables, map, moves)."""
    rows, width = tables.shape
    n = []
    for r in range(rows):
        m = int(lengths[r])
        n.append(-(-m // p))
        if not (0 <= m <= width * p and all(0 <= x < pages for x in tables[r, :n[r]])):
            return [INVALID, 0, 0, r], None, None, []
    live = sorted({int(x) for r in range(rows) for x in tables[r, :n[r]]})
    stay = set() if held is None else {x for x in range(pages) if held[x]}
    movable = [x for x in live if x not in stay]
    low = [x for x in range(pages) if x not in stay][:len(movable)]
    holes = sorted(set(low) - set(movable))
    moves = list(zip(sorted(set(movable) - set(low)), holes))
    to = np.full(pages, -1, np.int32)
    for x in live:
        to[x] = x
    for a, b in moves:
        to[a] = b
    out = np.full_like(tables, -1)
    for r in range(rows):
        out[r, :n[r]] = to[tables[r, :n[r]]]
    top = max([int(to.max()), *stay], default=-1) + 1
    return [0, top, len(moves), -1], out, to, moves


def sample(logits, mask, q_ln2, q_b, q_c, top_k, top_p, min_p, random):
    """(token, weight, total) of one row."""
    v = len(logits)
    w0 = q_b * q_b + q_c
    if not (1 <= q_ln2 <= 2 * q_b + 1 and q_b >= 0 and q_c >= 0 and 1 <= w0 <= 1 << 47 and w0 * v < 1 << 62 and top_k >= 0 and
            0 <= top_p <= 65536 and 0 <= min_p <= 65536):
        return -2, 0, 0
    legal = np.arange(v) if mask is None else np.nonzero(np.unpackbits(mask, bitorder="little")[:v])[0]
    if not len(legal):
        return -1, 0, 0
    x = logits[legal].astype(np.int64)
    order = np.lexsort((legal, -x))
    legal, d = legal[order], x[order][0] - x[order]
    z = d // q_ln2
    base = q_b - d % q_ln2
    w = np.where(z < 30, (base * base + q_c) >> np.minimum(z, 30), 0)
    if top_k:
        w = w[:top_k]
    run = np.cumsum(w)
    goal = -(-int(run[-1]) * top_p // 65536)
    w = w[:max(1, int(np.searchsorted(run, goal, "left")) + 1)]
    w = np.where(w >= -(-w0 * min_p // 65536), w, 0)
    run = np.cumsum(w)
    total = int(run[-1])
    at = int(np.searchsorted(run, total * random >> 32, "right"))
    return int(legal[at]), int(w[at]), total
