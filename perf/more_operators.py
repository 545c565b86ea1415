"""The operators of a server that gives several answers to a request, in plain form and as the framework's
kernels, for timing and comparing both.

* "update": pages of a cache change hands: contexts are forked, shortened, extended and freed, and a page that
  a row will write into while another row holds it is copied.
* "compact": the pages in use move to the lowest numbers.
* "store": new q, k and v rows: q and k rotated, k and v landed in pages of 8-bit codes with a scale, a power
  of two, per page, KV head and K or V.  A page's scale grows with its tokens, as if they came one by one.
* "attention": single tokens or chunks over such pages: integer scores, the i-exp softmax with Q15
  probabilities, P.V, the per-head context fold and the requant funnel over the row.
* "sample": the next token by temperature, top-k, top-p and min-p from given random numbers.

Everything is computed in integers, so both forms give the same bits.
"""
import numpy as np
import torch

own = False

# the i-exp's constants in Q30: ln 2, and b and c / a of exp(x) ~ a ((x + b)^2 + c / a) on (-ln 2, 0]
LN2, B, CA = 0.6931471805599453, 1.353, 0.344 / 0.3585
LN2_Q, B_Q, CA_Q = (int(x * 2 ** 30) for x in (LN2, B, CA))
SITE = (1518500250, -45)
MAX_SHIFT, MAX_VALUE = 8, 127 << 8  # the largest exponent of a page, the largest value it holds


def _named(name, case):
    return {"name": name, **case} if name else case


def _update(name, rows, group, tokens, page, layers, kv_heads, dim, table, fresh):
    """Groups of rows that share a context's first pages; `fresh`: only the first row of a group holds one yet."""
    return _named(name, {"kind": "update", "rows": rows, "group": group, "tokens": tokens, "page": page, "layers": layers,
                         "kv_heads": kv_heads, "dim": dim, "table": table, "fresh": fresh})


def _compact(name, rows, tokens, page, layers, kv_heads, dim, spare):
    return _named(name, {"kind": "compact", "rows": rows, "tokens": tokens, "page": page, "layers": layers,
                         "kv_heads": kv_heads, "dim": dim, "spare": spare})


def _store(name, rows, heads, kv_heads, dim, page, new, start, rotary, halves):
    return _named(name, {"kind": "store", "rows": rows, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
                         "new": new, "start": start, "rotary": rotary, "halves": halves})


def _attention(name, rows, heads, kv_heads, dim, page, new, lo, hi):
    return _named(name, {"kind": "attention", "rows": rows, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
                         "new": new, "lo": lo, "hi": hi})


def _sample(name, rows, vocab, masked):
    return _named(name, {"kind": "sample", "rows": rows, "vocab": vocab, "masked": masked})


def listed():
    return [
        # one chat of 350 tokens continued four ways: its open page is copied three times (all 28 layers of a 1.5B)
        _update("fork_4x350", 4, 4, 350, 64, 28, 2, 128, 32, True),
        # a step of 16 beams over each of 8 prompts: branches dropped and continued from each other (0.5B)
        _update("beams_128x1000", 128, 16, 1000, 64, 24, 2, 64, 64, False),
        # a small pool after a few chats have ended
        _compact("compact_6x200", 6, 200, 32, 28, 2, 128, 60),
        # a server's pool before part of it is given back (0.5B)
        _compact("compact_100x500", 100, 500, 64, 24, 2, 64, 900),
        # one token for each of 8 chats, somewhere inside their pages (1.5B, the framework's pair layout)
        _store("store_8x1", 8, 12, 2, 128, 64, 1, 777, 128, False),
        # prompts of several requests in one chunk (7B heads, half layout)
        _store("store_4x512", 4, 28, 4, 128, 64, 512, 0, 128, True),
        # two chats a few tokens in: latency
        _attention("attn_2x100", 2, 12, 2, 128, 64, 1, 90, 105),
        # a server's ordinary step: 24 requests of all lengths, small pages (1.5B)
        _attention("attn_24x1500", 24, 12, 2, 128, 32, 1, 1, 1500),
        # a full batch of long contexts (7B heads)
        _attention("attn_64x8000", 64, 28, 4, 128, 64, 1, 1000, 8000),
        # a long prompt's next chunk (1.5B)
        _attention("attn_chunk_500_at_2000", 1, 12, 2, 128, 64, 500, 2500, 2500),
        # one request over the full vocabulary
        _sample("sample_1x151936", 1, 151936, 0),
        # a large batch, every fourth row by another rule, half of them under a grammar
        _sample("sample_128x151936", 128, 151936, 64),
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))

    tops = {}
    for c in listed():
        w = work(c)
        tops[c["kind"]] = {k: max(w[k], tops.get(c["kind"], w)[k]) for k in w}
    while True:
        kind = rng.choice(["update", "compact", "store", "attention", "attention", "sample", "sample"])
        kv, dim, layers = rng.choice([(2, 128, 28), (2, 64, 24), (4, 128, 4), (1, 64, 3), (3, 32, 2)])
        page = rng.choice([16, 32, 64, 64, 128])
        if kind == "update":
            group, n = log(1, 16), log(1, 12)
            case = _update(None, group * n, group, log(1, 1500), page, layers, kv, dim, 1600 // page + rng.randrange(3, 9),
                           rng.random() < 0.5)
        elif kind == "compact":
            case = _compact(None, log(1, 128), log(1, 1200), page, layers, kv, dim, log(1, 900))
        elif kind == "store":
            heads, kv, dim = rng.choice([(12, 2, 128), (28, 4, 128), (14, 2, 64), (8, 2, 256), (4, 1, 32)])
            new = rng.choice([1, 1, log(2, 600)])
            start = rng.randrange(0, 2000) if new == 1 else page * rng.randrange(0, 1 + 2000 // page)
            case = _store(None, log(1, 128) if new == 1 else log(1, 6), heads, kv, dim, page, new, start,
                          rng.choice([dim, dim, dim // 2, dim // 4]), rng.random() < 0.5)
        elif kind == "attention":
            heads, kv, dim = rng.choice([(12, 2, 128), (12, 2, 128), (28, 4, 128), (14, 2, 64), (8, 2, 256), (4, 1, 32), (20, 1, 64)])
            new = rng.choice([1, 1, 1, log(2, 500)])
            hi = max(new, log(2, 12000))
            case = _attention(None, log(1, 96) if new == 1 else log(1, 4), heads, kv, dim, page, new, rng.randrange(new, hi + 1), hi)
        else:
            rows = log(1, 160)
            case = _sample(None, rows, log(300, 151936), rng.randrange(0, rows + 1))
        w = work(case)
        if all(w[k] <= tops[kind][k] for k in w) and w["bytes"] * (dim if kind == "attention" and case["new"] > 1 else 1) < 1 << 36:
            return case


# ---- inputs ----
def _random(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _codes(g, *shape):
    return torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda", generator=g)


def _bell(g, *shape):
    """Codes as the requant funnel leaves them: a bell with its largest at 127."""
    return (torch.randn(shape, device="cuda", generator=g) * 35.0).round_().clamp_(-127, 127).to(torch.int8)


def _mults(g, *shape):
    return torch.randint(1 << 30, 1 << 31, shape, dtype=torch.int64, device="cuda", generator=g).to(torch.int32)


def _scales(g, n, lo, hi):
    """Carried scales (m, e), value m 2^e, spread over [lo, hi] by their logarithm."""
    value = lo * (hi / lo) ** torch.rand(n, dtype=torch.float64, device="cuda", generator=g)
    part, e = torch.frexp(value)
    return torch.stack([(part * 2.0 ** 31).to(torch.int64), e.to(torch.int64) - 31], 1)


def _page_bytes(case):
    """(codes of K or V of a layer, a layer's, a page's): K, V, then the exponents."""
    half = case["kv_heads"] * case["page"] * case["dim"]
    layer = (2 * half + 2 * case["kv_heads"] + 15) // 16 * 16
    return half, layer, layer * case.get("layers", 1)


def _pages_of(n, page):
    return -(-n // page)


def _contexts(case):
    """The tables before an update: per row its pages and length.  A group's rows share all full pages of the first
    two thirds of its context."""
    rows, p = case["rows"], case["page"]
    tables, lengths, used = [], [], 0
    for r in range(rows):
        g, i = divmod(r, case["group"])
        n = max(1, case["tokens"] - 37 * g % max(1, case["tokens"]) - (i * 7919) % max(1, case["tokens"] // 4 + 1))
        if case["fresh"] and i:
            tables.append([])
            lengths.append(0)
            continue
        common = tables[r - i][:min(n // p, 2 * lengths[r - i] // 3 // p)] if i else []
        more = _pages_of(n, p) - len(common)
        tables.append(common + list(range(used, used + more)))
        used += more
        lengths.append(n)
    return tables, lengths, used


def _update_sources(case, lengths):
    """What each row becomes: (source, keep, room).  Beams continue themselves or another of their group; one in
    nine ends, one in eleven is cut back."""
    rows, group, out = case["rows"], case["group"], []
    for r in range(rows):
        g, i = divmod(r, group)
        if case["fresh"]:
            s = g * group
        else:
            s = g * group + (i if r * 2654435761 % 7 < 4 else r * 40503 % group)
        keep = lengths[s]
        if not case["fresh"] and r % 11 == 5:
            keep = keep * 2 // 3
        grow = 1 if not case["fresh"] else 1 + r * 13 % 40
        out.append((s, keep, keep + grow) if case["fresh"] or r % 9 != 4 else (-1, 0, 0))
    return out


def _update_counts(case):
    """(pages copied, pages of the pool) of an update."""
    p = case["page"]
    tables, lengths, used = _contexts(case)
    src = _update_sources(case, lengths)
    kept = [tables[s][:_pages_of(k, p)] if s >= 0 else [] for s, k, _ in src]
    tails = [t[-1] if k % p and n > k else -1 for t, (_, k, n) in zip(kept, src)]
    every, growing = {}, {}
    for t, tail in zip(kept, tails):
        for x in t:
            every[x] = every.get(x, 0) + 1
        if tail >= 0:
            growing[tail] = growing.get(tail, 0) + 1
    copied = sum(n if every[x] > n else n - 1 for x, n in growing.items())
    return copied, used + case["rows"] * 2 + sum(_pages_of(n, p) - _pages_of(k, p) for _, k, n in src)


def _compact_lengths(case):
    return [max(1, case["tokens"] - (r * 7919) % (case["tokens"] // 2 + 1)) for r in range(case["rows"])]


def _compact_pages(case):
    """The rows' pages, spread over a pool with `spare` more: every page in a random place."""
    need = sum(_pages_of(n, case["page"]) for n in _compact_lengths(case))
    return need, need + case["spare"]


def _tables(case, lists, width, perm):
    out = np.full((len(lists), width), -1, np.int32)
    for r, t in enumerate(lists):
        out[r, :len(t)] = perm[t]
    return torch.from_numpy(out).cuda()


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _i64(x):
    return torch.tensor(x, dtype=torch.int64, device="cuda")


def _pool(g, pages, nbytes):
    pool = torch.empty((pages, nbytes), dtype=torch.int8, device="cuda")
    return pool.random_(-127, 128, generator=g)


def _prepare_update(case, seed):
    g, nbytes = _random(seed), _page_bytes(case)[2]
    tables, lengths, _ = _contexts(case)
    pages = _update_counts(case)[1]
    perm = np.random.default_rng(seed).permutation(pages).astype(np.int32)
    src = _update_sources(case, lengths)
    t = _tables(case, tables, case["table"], perm)
    return {"case": case, "pool": _pool(g, pages, nbytes), "tables": t, "lengths": _i64(lengths),
            "source": _i32([s for s, _, _ in src]), "keep": _i64([k for _, k, _ in src]), "room": _i64([n for _, _, n in src]),
            "new_tables": torch.zeros_like(t), "new_lengths": torch.zeros(case["rows"], dtype=torch.int64, device="cuda"),
            "result": torch.zeros(4, dtype=torch.int32, device="cuda")}


def _prepare_compact(case, seed):
    g, nbytes = _random(seed), _page_bytes(case)[2]
    lengths = _compact_lengths(case)
    need, pages = _compact_pages(case)
    perm = np.random.default_rng(seed).permutation(pages).astype(np.int32)
    ends = np.cumsum([_pages_of(n, case["page"]) for n in lengths])
    lists = [list(range(b - _pages_of(n, case["page"]), b)) for n, b in zip(lengths, ends)]
    t = _tables(case, lists, max(map(len, lists)) + 2, perm)
    held = torch.zeros(pages, dtype=torch.uint8, device="cuda")
    held[torch.from_numpy(perm[need::13].astype(np.int64)).cuda()] = 1  # pages that another part of the server keeps
    return {"case": case, "pool": _pool(g, pages, nbytes), "tables": t, "lengths": _i64(lengths), "held": held,
            "new_tables": torch.zeros_like(t), "map": torch.zeros(pages, dtype=torch.int32, device="cuda"),
            "result": torch.zeros(4, dtype=torch.int32, device="cuda")}


def _row_counts(case):
    """(first position, new tokens) per row: chunks end at different places."""
    out = []
    for r in range(case["rows"]):
        n = case["new"] - (r * 7919) % (case["new"] // 3 + 1)
        if case["kind"] == "store":
            out.append((case["start"] + (0 if case["new"] > 1 else r * 7919 % 61), n))
        else:
            end = case["lo"] + (r * 7919 + case["hi"] - case["lo"]) % (case["hi"] - case["lo"] + 1)
            out.append((max(0, end - n), min(n, end)))
    return out


def _prepare_rows(case, seed, shift_lo, shift_hi):
    """Pages, tables and the rows' tokens, alike for the store and the attention."""
    g, p = _random(seed), case["page"]
    rows, half, nbytes = _row_counts(case), *_page_bytes(case)[::2]
    lists, used = [], 0
    for s, n in rows:
        m = _pages_of(s + n, p)
        lists.append(list(range(used, used + m)))
        used += m
    pages = used + 1 + used // 16
    perm = np.random.default_rng(seed).permutation(pages).astype(np.int32)
    pool = _pool(g, pages, nbytes)
    kv = case["kv_heads"]
    pool[:, 2 * half:2 * half + 2 * kv] = torch.randint(shift_lo, shift_hi + 1, (pages, 2 * kv), dtype=torch.int8, device="cuda", generator=g)
    cuts = [0] + np.cumsum([n for _, n in rows]).tolist()
    return g, {"case": case, "pool": pool, "tables": _tables(case, lists, max(map(len, lists)), perm), "row_tokens": _i32(cuts),
               "row_start": _i64([s for s, _ in rows]), "tokens": cuts[-1], "max_new": max(n for _, n in rows),
               "max_width": max(s + n for s, n in rows)}


def _prepare_store(case, seed):
    # pages met half full hold values of a middling size: new tokens make some of them grow
    g, s = _prepare_rows(case, seed, 2, 4)
    t, nh, nkv, d = s["tokens"], case["heads"], case["kv_heads"], case["dim"]
    pairs, top = case["rotary"] // 2, s["max_width"]
    angle = torch.arange(top, dtype=torch.float64, device="cuda")[:, None] * 1e6 ** (-torch.arange(pairs, dtype=torch.float64, device="cuda") / pairs)
    s |= {"cos": (angle.cos() * 2 ** 30).round().to(torch.int64), "sin": (angle.sin() * 2 ** 30).round().to(torch.int64)}
    # a unit of the cache is about a sixteenth of an ordinary code
    unit = _scales(g, 2 * nkv, 0.9e-3, 1.4e-3)
    recip = torch.tensor([((1 << 63) + m) // (2 * m) for m in unit[:, 0].tolist()], dtype=torch.int64, device="cuda")
    s |= {"q": _bell(g, t, nh * d), "k": _bell(g, t, nkv * d), "v": _bell(g, t, nkv * d), "k_scale": _scales(g, t, 0.004, 0.06),
          "v_scale": _scales(g, t, 0.002, 0.05), "r_k": recip[:nkv].clone(), "r_v": recip[nkv:].clone(),
          "e_k": unit[:nkv, 1].clone(), "e_v": unit[nkv:, 1].clone(),
          "q_out": torch.zeros((t, nh * d), dtype=torch.int8, device="cuda"),
          "clamped": torch.zeros(case["rows"], dtype=torch.int32, device="cuda"),
          "status": torch.zeros(case["rows"], dtype=torch.int32, device="cuda")}
    return s


def _prepare_attention(case, seed):
    g, s = _prepare_rows(case, seed, 2, 4)
    t, nh, nkv, d = s["tokens"], case["heads"], case["kv_heads"], case["dim"]
    fold = torch.zeros((nh, 3), dtype=torch.int32, device="cuda")
    fold[:, 1] = _mults(g, nh)
    fold[:, 2] = torch.randint(2, 6, (nh,), device="cuda", generator=g)
    khead = _scales(g, nkv, 0.1 / 127 / d ** 0.5, 0.2 / 127 / d ** 0.5)
    s |= {"q": _codes(g, t, nh * d), "q_scale": _scales(g, t, 1.0 / 127, 6.0 / 127), "khead_m": khead[:, 0].clone(),
          "khead_e": khead[:, 1].clone(), "fold": fold, "codes": torch.zeros((t, nh * d), dtype=torch.int8, device="cuda"),
          "scales": torch.zeros((t, 2), dtype=torch.int64, device="cuda"),
          "status": torch.zeros(t, dtype=torch.int32, device="cuda")}
    return s


def _prepare_sample(case, seed):
    g, rows, v = _random(seed), case["rows"], case["vocab"]
    # logits of an integer head: a bell of some 10^5 units, whose largest stands out in some rows
    logits = (torch.randn((rows, v), device="cuda", generator=g) * 120000.0).to(torch.int32)
    logits[::3, ::997] += 150000
    page = (v + 7) // 8
    mask = torch.randint(0, 256, (rows, page), dtype=torch.uint8, device="cuda", generator=g)
    mask &= torch.randint(0, 256, (rows, page), dtype=torch.uint8, device="cuda", generator=g)
    host = np.random.default_rng(seed)
    unit = host.uniform(0.6, 1.4, rows) * 45000.0  # logit units of one, by each request's temperature
    rule = np.zeros((rows, 7), np.int64)  # q_ln2, q_b, q_c, top_k, top_p, min_p, random
    rule[:, 0], rule[:, 1], rule[:, 2] = (LN2 * unit).astype(np.int64), (B * unit).astype(np.int64), (CA * unit * unit).astype(np.int64)
    form = np.arange(rows) % 4  # top-k and top-p, as most requests have them; top-p alone; all three; temperature alone
    rule[:, 3] = np.where(form == 0, host.integers(20, 60, rows), np.where(form == 2, host.integers(100, 400, rows), 0))
    rule[:, 4] = np.where(form == 3, 65536, host.integers(52000, 64000, rows))
    rule[:, 5] = np.where(form == 2, host.integers(600, 6000, rows), 0)
    rule[:, 6] = host.integers(0, 1 << 32, rows)
    table = np.zeros((rows, 6), np.int64)  # the records that a program keeps on the device
    small = table.view(np.uint32).reshape(rows, 12)
    table[:, 0] = [mask[r].data_ptr() if r < case["masked"] else 0 for r in range(rows)]
    table[:, 1:4], small[:, 8:12] = rule[:, :3], rule[:, 3:]
    return {"case": case, "logits": logits, "mask": mask, "rule": torch.from_numpy(rule).cuda(), "table": torch.from_numpy(table).cuda(),
            "picked": torch.zeros(rows, dtype=torch.int32, device="cuda"), "mass": torch.zeros((rows, 2), dtype=torch.int64, device="cuda")}


def prepare(case, seed):
    return {"update": _prepare_update, "compact": _prepare_compact, "store": _prepare_store, "attention": _prepare_attention,
            "sample": _prepare_sample}[case["kind"]](case, seed)


# ---- what a pass cannot do without ----
def work(case):
    if case["kind"] == "update":
        copied, pages = _update_counts(case)
        cells = case["rows"] * case["table"]
        return {"bytes": 2 * copied * _page_bytes(case)[2] + 8 * cells + 40 * case["rows"], "flops": 2 * cells + pages}
    if case["kind"] == "compact":
        need, pages = _compact_pages(case)
        held = len(range(need, pages, 13))
        # of `need` pages in random places, those that lie past the first `need` that nobody keeps
        moved = need * (pages - held - need) / max(1, pages - held)
        return {"bytes": 2 * moved * _page_bytes(case)[2] + 8 * need + 5 * pages, "flops": 2 * need + pages}
    if case["kind"] == "sample":
        rows, v = case["rows"], case["vocab"]
        return {"bytes": 4 * rows * v + case["masked"] * ((v + 7) // 8) + 68 * rows, "flops": 8 * rows * v}
    rows, nh, nkv, d = _row_counts(case), case["heads"], case["kv_heads"], case["dim"]
    t = sum(n for _, n in rows)
    if case["kind"] == "store":
        return {"bytes": t * (2 * nh * d + 4 * nkv * d + 32) + 16 * (case["rotary"] // 2) * max(n for _, n in rows),
                "flops": t * (6 * nh * d + 12 * nkv * d)}
    reach = sum(n * s + n * (n + 1) // 2 for s, n in rows)
    return {"bytes": sum(s + n for s, n in rows) * 2 * nkv * d + t * (2 * nh * d + 52), "flops": 4 * nh * d * reach}


# ---- the plain form ----
def _srdhm(a, b):
    return (a * b + (1 << 30)) >> 31


def _shift_away(x, e):
    """x / 2^e, ties away from zero."""
    mask = (torch.ones_like(x) << e) - 1
    return (x >> e) + ((x & mask) > (mask >> 1) + (x < 0)).to(torch.int64)


def _combine(m1, e1, m2, e2):
    m, e = _srdhm(m1, m2), e1 + e2 + 31
    low = m < (1 << 30)
    return torch.where(low, m << 1, m), e - low.to(torch.int64)


def _reciprocal(m):
    """2^62 / m to the nearest, for m in [2^30, 2^31)."""
    y = (1 << 62) // m
    return y + (2 * ((1 << 62) - y * m) >= m).to(torch.int64)


def _funnel(x, m, e):
    """The rows of x to codes in [-127, 127] and their scales, times the carried scale (m, e)."""
    ax = x.abs()
    d = ax.amax(1).clamp(min=1)
    s = 31 - torch.frexp(d.double())[1].to(torch.int64)
    dn = torch.where(s >= 0, d << s.clamp(min=0), d >> 1)
    f, shift = 127 * _reciprocal(dn)[:, None], (62 - s)[:, None]
    high = ax * (f >> 16) + ((ax * (f & 0xffff)) >> 16)
    code = ((high + (torch.ones_like(shift) << (shift - 17))) >> (shift - 16)).clamp(max=127) * x.sign()
    return code.to(torch.int8), torch.stack(_combine(m, e, dn, -s), 1)


def _counts(lengths, page):
    return (lengths + page - 1) // page


def _plain_update(s):
    case, p, pool = s["case"], s["case"]["page"], s["pool"]
    rows, width, pages, dev = case["rows"], case["table"], s["pool"].shape[0], s["pool"].device
    src, keep, room = s["source"].long(), s["keep"], s["room"]
    cell, row = torch.arange(width, device=dev)[None], torch.arange(rows, device=dev)
    kept, need = _counts(keep, p), _counts(room, p)
    old = torch.where(cell < kept[:, None], s["tables"][src.clamp(min=0)].long(), -1)
    grows = (keep % p != 0) & (room > keep)
    tail = old.gather(1, (kept - 1).clamp(min=0)[:, None])[:, 0]
    refs = torch.zeros(pages + 1, dtype=torch.int64, device=dev).index_add_(0, (old + 1).flatten(), torch.ones_like(old.flatten()))[1:]
    at = torch.where(grows, tail, pages)
    grown = torch.zeros(pages + 1, dtype=torch.int64, device=dev).index_add_(0, at, torch.ones_like(at))[:pages]
    lowest = torch.full((pages + 1,), rows, dtype=torch.int64, device=dev).scatter_reduce_(0, at, row, "amin")[:pages]
    t = tail.clamp(min=0)
    copies = grows & ((refs[t] > grown[t]) | (lowest[t] < row))
    free = (refs == 0).nonzero()[:, 0]
    wants = copies.long() + need - kept
    first = wants.cumsum(0) - wants
    # a row's free pages: its copy's first, then those past what it kept
    i = torch.where(cell >= kept[:, None], cell - kept[:, None] + copies[:, None].long(), 0) + first[:, None]
    given = free[i.clamp(max=max(0, len(free) - 1))]
    fresh = ((cell >= kept[:, None]) & (cell < need[:, None])) | (copies[:, None] & (cell == kept[:, None] - 1))
    s["new_tables"].copy_(torch.where(fresh, given, old))
    s["new_lengths"].copy_(room)
    to = free[first.clamp(max=max(0, len(free) - 1))]
    pool[to[copies]] = pool[tail[copies]]
    nothing = torch.zeros((), dtype=torch.int64, device=dev)
    s["result"].copy_(torch.stack([nothing, len(free) - wants.sum(), copies.sum(), nothing - 1]))
    return {"tables": s["new_tables"], "lengths": s["new_lengths"], "result": s["result"], "pool": pool}


def _plain_compact(s):
    case, pool, dev = s["case"], s["pool"], s["pool"].device
    pages, old = pool.shape[0], s["tables"].long()
    mine = torch.arange(old.shape[1], device=dev)[None] < _counts(s["lengths"], case["page"])[:, None]
    live = torch.zeros(pages + 1, dtype=torch.bool, device=dev).index_fill_(0, torch.where(mine, old, pages).flatten(), True)[:pages]
    index, held = torch.arange(pages, device=dev), s["held"] != 0
    movable, rank = live & ~held, (~held).long().cumsum(0)  # rank: how many pages up to here nobody keeps
    inside = rank <= movable.sum()
    moved, holes = (movable & ~inside).nonzero()[:, 0], (~held & ~live & inside).nonzero()[:, 0]
    to = torch.where(live, index, -1)
    to[moved] = holes
    s["map"].copy_(to)
    s["new_tables"].copy_(torch.where(mine, to[old.clamp(min=0)], -1))
    pool[holes] = pool[moved]
    nothing = torch.zeros((), dtype=torch.int64, device=dev)
    last = torch.where((to >= 0) | held, torch.where(to >= 0, to, index), -1).amax() + 1
    s["result"].copy_(torch.stack([nothing, last, torch.full_like(nothing, len(moved)), nothing - 1]))
    return {"tables": s["new_tables"], "map": s["map"], "result": s["result"], "pool": pool}


def _rotate(x, cos, sin, halves):
    """x [tokens, heads, dim] in 64 bits; the first 2 * pairs of each head turn."""
    pairs = cos.shape[1]
    a, rest = x[..., :2 * pairs], x[..., 2 * pairs:]
    u, v = (a[..., :pairs], a[..., pairs:]) if halves else (a[..., ::2], a[..., 1::2])
    c, n = cos[:, None], sin[:, None]
    u, v = _shift_away(u * c - v * n, 30), _shift_away(u * n + v * c, 30)
    return torch.cat([torch.cat([u, v], 2) if halves else torch.stack([u, v], 3).flatten(2), rest], 2)


def _landed(code, scale, recip, e_unit):
    """round(code m recip / 2^k) with ties away from zero; the product passes 2^63."""
    am = code.abs() * scale[:, :1, None]
    k = 62 - (scale[:, 1, None] - e_unit[None])
    r = recip[None, :, None]
    high = am * (r >> 16) + ((am * (r & 0xffff)) >> 16)
    k = k[:, :, None]
    return ((high + (torch.ones_like(k) << (k - 17))) >> (k - 16)) * code.sign()


def _limits(dev):
    """The largest value that an exponent of 0, 1, ... holds in 8 bits."""
    return torch.tensor([127] + [(255 << (e - 1)) - 1 for e in range(1, MAX_SHIFT)], device=dev)


def _plain_store(s):
    case, dev = s["case"], s["pool"].device
    p, nkv, d, rows = case["page"], case["kv_heads"], case["dim"], case["rows"]
    cuts, start, half = s["row_tokens"].long(), s["row_start"], _page_bytes(case)[0]
    row = torch.repeat_interleave(torch.arange(rows, device=dev), cuts.diff(), output_size=s["tokens"])
    pos = start[row] + torch.arange(s["tokens"], device=dev) - cuts[row]
    cos, sin = s["cos"][pos], s["sin"][pos]
    q = _rotate(s["q"].view(s["tokens"], -1, d).to(torch.int64), cos, sin, case["halves"])
    s["q_out"].copy_(q.clamp(-127, 127).view(s["tokens"], -1))
    k, v = (_landed(s[x].view(-1, nkv, d).to(torch.int64), s[x + "_scale"], s["r_" + x], s["e_" + x]) for x in "kv")
    clamped = (k.abs() > MAX_VALUE).sum((1, 2)) + (v.abs() > MAX_VALUE).sum((1, 2))
    k = _rotate(k.clamp(-MAX_VALUE, MAX_VALUE), cos, sin, case["halves"])
    clamped = clamped + (k.abs() > MAX_VALUE).sum((1, 2))
    s["clamped"].copy_(torch.zeros(rows, dtype=torch.int64, device=dev).index_add_(0, row, clamped))
    x = torch.stack([k, v.clamp(-MAX_VALUE, MAX_VALUE)], 1).clamp(-MAX_VALUE, MAX_VALUE)  # [tokens, K | V, head, dim]
    # the pages that the rows touch, one grid of slots; those before a row's first token hold codes already
    most = (s["max_new"] + p - 2) // p + 1
    at = start // p
    slot = (pos // p - at[row]) * p + pos % p
    cell = torch.arange(most, device=dev)
    touched = cell[None] <= (start + cuts.diff() - 1)[:, None] // p - at[:, None]
    page = s["tables"].long().gather(1, (at[:, None] + cell).clamp(max=s["tables"].shape[1] - 1))
    grid = s["pool"][page][..., :2 * half].view(rows, most, 2, nkv, p, d).to(torch.int64)
    exps = s["pool"][page][..., 2 * half:2 * half + 2 * nkv].view(rows, most, 2, nkv).to(torch.int64)
    there = (cell[None, :, None] * p + torch.arange(p, device=dev)) < (start % p)[:, None, None]  # [rows, most, slot]
    level = torch.where(there[:, :, None, None], exps[..., None], 0)
    flat = (row, slot // p, slice(None), slice(None), slot % p)
    need = (x.abs().amax(3, keepdim=True) > _limits(dev)).sum(3)
    level[flat] = need
    fresh = torch.zeros((rows, most, 1, 1, p), dtype=torch.bool, device=dev)
    fresh[row, slot // p, 0, 0, slot % p] = True
    level = level.cummax(4)[0]
    value = grid.clone()
    value[flat] = _shift_away(x, level[flat][..., None])
    reached = level.clone()
    for e in range(1, MAX_SHIFT + 1):  # codes are rounded once more at each exponent that their page reaches after them
        grows = (fresh & (level == e)).any(4, keepdim=True) & (reached < e)
        value = torch.where(grows[..., None], _shift_away(value, (e - reached).clamp(min=0)[..., None]), value)
        reached = torch.where(grows, e, reached)
    live = there[:, :, None, None] | fresh
    grid = torch.where(live[..., None], value, grid)
    out = s["pool"][page]
    out[..., :2 * half] = grid.view(rows, most, 2 * half).to(torch.int8)
    out[..., 2 * half:2 * half + 2 * nkv] = torch.where(live, level, 0).amax(4).view(rows, most, 2 * nkv).to(torch.int8)
    s["pool"][page[touched]] = out[touched]
    s["status"].zero_()
    return {"pool": s["pool"], "q": s["q_out"], "clamped": s["clamped"], "status": s["status"]}


def _plain_attention(s):
    case, dev = s["case"], s["pool"].device
    rows, nh, nkv, d, p = (case[x] for x in ("rows", "heads", "kv_heads", "dim", "page"))
    grp, new, t = nh // nkv, s["max_new"], s["tokens"]
    cuts, start, half, wide = s["row_tokens"].long(), s["row_start"], _page_bytes(case)[0], s["max_width"]
    row = torch.repeat_interleave(torch.arange(rows, device=dev), cuts.diff(), output_size=t)
    at = torch.arange(t, device=dev) - cuts[row]
    # the softmax's integer constants per (token, kv head), from the scale of one unit of score
    sm, se = _combine(s["q_scale"][:, :1], s["q_scale"][:, 1:], s["khead_m"][None], s["khead_e"][None])
    r = _reciprocal(sm)
    q_ln2, q_b = (LN2_Q * r) >> (92 + se), (B_Q * r) >> (92 + se)
    ca = CA_Q * r
    q_c = (r * (ca >> 31) + ((r * (ca & 0x7fffffff)) >> 31)) >> (123 + 2 * se)

    def grid(x, rest):  # [tokens, kv, ...] to [rows, kv, new, ...]
        out = torch.zeros((rows, new, nkv) + rest, dtype=x.dtype, device=dev)
        out[row, at] = x
        return out.transpose(1, 2)

    q = grid(s["q"].reshape(t, nkv, grp, d).float(), (grp, d)).reshape(rows, nkv, new * grp, d)
    q_ln2, q_b, q_c = (grid(x, ())[..., None, None] for x in (q_ln2.clamp(min=1), q_b, q_c))
    q_ln2 = q_ln2.clamp(min=1)
    page = s["tables"].long().clamp(min=0)  # positions past a row's end are masked below
    kv = s["pool"][page]
    kc, vc = (kv[..., i * half:(i + 1) * half].reshape(rows, -1, nkv, p, d).transpose(1, 2).reshape(rows, nkv, -1, d)[:, :, :wide].float() for i in (0, 1))
    exps = kv[..., 2 * half:2 * half + 2 * nkv].reshape(rows, -1, 2, nkv).to(torch.int64).permute(2, 0, 3, 1)
    ks, vs = exps.repeat_interleave(p, dim=3)[..., :wide]
    score = torch.matmul(q, kc.transpose(2, 3).contiguous()).to(torch.int64) << ks[:, :, None]
    score = score.reshape(rows, nkv, new, grp, wide)
    end = start[:, None] + torch.arange(new, device=dev) + 1
    live = (torch.arange(wide, device=dev) < end[..., None])[:, None, :, None]
    top = torch.where(live, score, -(1 << 40)).amax(4, keepdim=True)
    x = torch.minimum(top - score, 30 * q_ln2).clamp(min=0)
    z = x // q_ln2
    base = q_b - (x - z * q_ln2)
    e = torch.where(live, (base * base + q_c) >> z, 0)
    prob = ((e << 15) // e.sum(4, keepdim=True).clamp(min=1)).double().reshape(rows, nkv, new * grp, wide)
    # at most 2^15 times 127 2^8 in all: exact in 64-bit floats
    ctx = torch.matmul(prob, vc.double() * torch.exp2(vs.double())[..., None])
    ctx = ctx.to(torch.int64).reshape(rows, nkv, new, grp, d).transpose(1, 2)[row, at].reshape(t, nh, d)
    fold = s["fold"].to(torch.int64)
    x = _shift_away(_srdhm(ctx, fold[:, 1, None]), fold[:, 2, None]).reshape(t, nh * d)
    site = torch.tensor(SITE, dtype=torch.int64, device=dev)
    codes, scales = _funnel(x, site[0].expand(t), site[1].expand(t))
    return {"codes": codes, "scales": scales, "status": torch.zeros(t, dtype=torch.int32, device=dev)}


def _plain_sample(s):
    case, rule, dev = s["case"], s["rule"], s["logits"].device
    rows, v = case["rows"], case["vocab"]
    bits = ((s["mask"][:, :, None] >> torch.arange(8, dtype=torch.uint8, device=dev)) & 1).view(rows, -1)[:, :v].bool()
    legal = bits | (torch.arange(rows, device=dev) >= case["masked"])[:, None]
    x = torch.where(legal, s["logits"].to(torch.int64), -(1 << 40))
    x, index = torch.sort(x, dim=1, descending=True, stable=True)  # equal logits by the lower index
    q_ln2, q_b, q_c, top_k, top_p, min_p, random = (rule[:, i, None] for i in range(7))
    d = x[:, :1] - x
    z = d // q_ln2
    base = q_b - (d - z * q_ln2)
    w = torch.where((x > -(1 << 40)) & (z < 30), (base * base + q_c) >> z.clamp(max=30), 0)
    place = torch.arange(v, device=dev)[None]
    w = torch.where((top_k == 0) | (place < top_k), w, 0)
    # the shortest run of the first ones with the share top_p of their sum
    run = w.cumsum(1)
    total = run[:, -1:]
    need = (total >> 16) * top_p + (((total & 0xffff) * top_p + 0xffff) >> 16)
    w = torch.where((place == 0) | (run - w < need), w, 0)
    w0 = q_b * q_b + q_c
    w = torch.where(w >= (w0 >> 16) * min_p + (((w0 & 0xffff) * min_p + 0xffff) >> 16), w, 0)
    run = w.cumsum(1)
    total = run[:, -1:]
    low = total & 0xffffffff  # its product with 32 bits passes 2^63
    target = (total >> 32) * random + ((low * (random >> 16) + ((low * (random & 0xffff)) >> 16)) >> 16)
    at = (run <= target).sum(1, keepdim=True).clamp(max=v - 1)
    some = legal.any(1)
    token = torch.where(some, index.gather(1, at)[:, 0], -1).to(torch.int32)
    mass = torch.where(some[:, None], torch.cat([w.gather(1, at), total], 1), 0)
    return {"tokens": token, "mass": mass}


# ---- the framework's operators ----
_LIB = []


def _ops():
    if not _LIB:
        import os

        from superslm_amd.batch_ops import BatchOps
        from superslm_amd.cache_ops import CacheOps
        from superslm_amd.sslm import SslmLib

        here = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        lib = SslmLib(os.path.join(here, "superslm_amd", "libsslm_hip.so"))
        _LIB.append((CacheOps(lib), BatchOps(lib)))
    return _LIB[0]


def _own_call(s):
    """The call over this state's buffers, with its workspace: made once, as a server's decode loop does."""
    case, (cache, batch) = s["case"], _ops()
    p = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}

    def space(n):
        s["workspace"] = torch.empty((n,), dtype=torch.uint8, device="cuda")
        return {"workspace": s["workspace"].data_ptr(), "workspace_bytes": n}

    if case["kind"] == "sample":
        shape = dict(rows=case["rows"], vocab=case["vocab"])
        return batch.sample_tokens(**shape, **space(batch.sample_workspace(**shape)), logits=p["logits"], rules=p["table"],
                                   tokens=p["picked"], mass=p["mass"])
    half, _, nbytes = _page_bytes(case)
    table = dict(rows=case["rows"], pages=s["pool"].shape[0], table_ld=s["tables"].shape[1])
    pool = dict(pool=p["pool"], page_bytes=nbytes, page_tokens=case["page"], tables=p["tables"])
    if case["kind"] == "update":
        return cache.update(**table, **pool, **space(cache.update_workspace(**table)), lengths=p["lengths"], source=p["source"],
                            keep=p["keep"], room=p["room"], new_tables=p["new_tables"], new_lengths=p["new_lengths"], result=p["result"])
    if case["kind"] == "compact":
        return cache.compact(**table, **pool, **space(cache.compact_workspace(**table)), lengths=p["lengths"], held=p["held"],
                             new_tables=p["new_tables"], map=p["map"], result=p["result"])
    rows = dict(rows=case["rows"], tokens=s["tokens"], heads=case["heads"], kv_heads=case["kv_heads"], head_dim=case["dim"],
                max_new=s["max_new"])
    pool |= dict(pages=table["pages"], table_ld=table["table_ld"], row_tokens=p["row_tokens"], row_start=p["row_start"],
                 k_offset=0, v_offset=half, exp_offset=2 * half)
    if case["kind"] == "store":
        return cache.store(**rows, **pool, rope_dim=case["rotary"], rope_halves=int(case["halves"]), rope_rows=s["max_width"],
                           rope_cos=p["cos"], rope_sin=p["sin"], q=p["q"], k=p["k"], v=p["v"], k_scale=p["k_scale"], v_scale=p["v_scale"],
                           r_t_k=p["r_k"], e_t_k=p["e_k"], r_t_v=p["r_v"], e_t_v=p["e_v"], q_out=p["q_out"], clamped=p["clamped"],
                           status=p["status"])
    shape = dict(rows, page_tokens=case["page"], max_width=s["max_width"])
    return cache.attention(**rows, **pool, max_width=s["max_width"], **space(cache.attention_workspace(**shape)), q=p["q"],
                           q_scale=p["q_scale"], khead_m=p["khead_m"], khead_e=p["khead_e"], ln2_q=LN2_Q, b_q=B_Q, ca_q=CA_Q,
                           ctx_fold=p["fold"], site=SITE, codes=p["codes"], scales=p["scales"], status=p["status"])


def run(state):
    kind = state["case"]["kind"]
    if not own:
        return {"update": _plain_update, "compact": _plain_compact, "store": _plain_store, "attention": _plain_attention,
                "sample": _plain_sample}[kind](state)
    if "call" not in state:
        state["call"] = _own_call(state)
    state["call"](torch.cuda.current_stream().cuda_stream)
    if kind == "update":
        return {"tables": state["new_tables"], "lengths": state["new_lengths"], "result": state["result"], "pool": state["pool"]}
    if kind == "compact":
        return {"tables": state["new_tables"], "map": state["map"], "result": state["result"], "pool": state["pool"]}
    if kind == "store":
        return {"pool": state["pool"], "q": state["q_out"], "clamped": state["clamped"], "status": state["status"]}
    if kind == "attention":
        return {"codes": state["codes"], "scales": state["scales"], "status": state["status"]}
    return {"tokens": state["picked"], "mass": state["mass"]}


# ---- from the definitions, on the host ----
def _host(s):
    return {k: x.cpu().numpy() for k, x in s.items() if isinstance(x, torch.Tensor)}


def _round_shift(x, e):
    half = (np.int64(1) << e) >> 1
    return np.sign(x) * ((np.abs(x) + half) >> e)


def _exact_update(case, s):
    h, p, rows = _host(s), case["page"], case["rows"]
    kept = [h["tables"][h["source"][r], :_pages_of(int(h["keep"][r]), p)].tolist() if h["source"][r] >= 0 else [] for r in range(rows)]
    writes = [bool(h["keep"][r] % p) and h["room"][r] > h["keep"][r] for r in range(rows)]
    holders = {}
    for r, t in enumerate(kept):
        for i, x in enumerate(t):
            holders.setdefault(x, []).append((r, writes[r] and i == len(t) - 1))
    free = [x for x in range(len(h["pool"])) if x not in holders]
    out, used, copied = np.full_like(h["tables"], -1), 0, 0
    for r, t in enumerate(kept):
        t = list(t)
        if writes[r]:
            others = [(q, w) for q, w in holders[t[-1]] if q != r]
            if any(not w or q < r for q, w in others):
                h["pool"][free[used]] = h["pool"][t[-1]]
                t[-1] = free[used]
                used, copied = used + 1, copied + 1
        while len(t) < _pages_of(int(h["room"][r]), p):
            t.append(free[used])
            used += 1
        out[r, :len(t)] = t
    return {"tables": out, "lengths": h["room"], "result": np.array([0, len(free) - used, copied, -1], np.int32), "pool": h["pool"]}


def _exact_compact(case, s):
    h, p = _host(s), case["page"]
    n = [_pages_of(int(x), p) for x in h["lengths"]]
    live = {int(x) for r, m in enumerate(n) for x in h["tables"][r, :m]}
    open_ = [x for x in range(len(h["pool"])) if not h["held"][x]]
    count = sum(not h["held"][x] for x in live)
    low = set(open_[:count])
    to = {x: x for x in live}
    to.update(zip(sorted(x for x in live if not h["held"][x] and x not in low), sorted(low - live)))
    moved = [(a, b) for a, b in to.items() if a != b]
    for a, b in moved:
        h["pool"][b] = h["pool"][a]
    out, table = np.full_like(h["map"], -1), np.full_like(h["tables"], -1)
    for a, b in to.items():
        out[a] = b
    for r, m in enumerate(n):
        table[r, :m] = out[h["tables"][r, :m]]
    top = max([*to.values(), *np.nonzero(h["held"])[0].tolist()], default=-1) + 1
    return {"tables": table, "map": out, "result": np.array([0, top, len(moved), -1], np.int32), "pool": h["pool"]}


def _turned(x, cos, sin, halves):
    y, pairs = x.copy(), len(cos)
    a, b = (slice(0, pairs), slice(pairs, 2 * pairs)) if halves else (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2))
    y[..., a], y[..., b] = _round_shift(x[..., a] * cos - x[..., b] * sin, 30), _round_shift(x[..., a] * sin + x[..., b] * cos, 30)
    return y


def _exact_store(case, s):
    h, p, nkv, d = _host(s), case["page"], case["kv_heads"], case["dim"]
    half, pool, q = _page_bytes(case)[0], h["pool"], np.zeros_like(h["q_out"])
    clamped = np.zeros_like(h["clamped"])
    for r in range(case["rows"]):
        for t in range(h["row_tokens"][r], h["row_tokens"][r + 1]):
            pos = int(h["row_start"][r]) + int(t - h["row_tokens"][r])
            cos, sin = h["cos"][pos], h["sin"][pos]
            q[t] = np.clip(_turned(h["q"][t].reshape(-1, d).astype(np.int64), cos, sin, case["halves"]), -127, 127).reshape(-1)
            for i, x in enumerate("kv"):
                m, e = (int(y) for y in h[x + "_scale"][t])
                # round(|code| m r / 2^k) by the code's magnitude: 128 values a head
                known = [[(2 * c * m * int(r_) + (1 << k)) >> (k + 1) for c in range(128)]
                         for r_, k in ((h["r_" + x][j], 62 - (e - int(h["e_" + x][j]))) for j in range(nkv))]
                code = h[x][t].reshape(nkv, d).astype(np.int64)
                y = np.take_along_axis(np.array(known), np.abs(code), 1) * np.sign(code)
                clamped[r] += int((np.abs(y) > MAX_VALUE).sum())
                y = np.clip(y, -MAX_VALUE, MAX_VALUE)
                if x == "k":
                    y = _turned(y, cos, sin, case["halves"])
                    clamped[r] += int((np.abs(y) > MAX_VALUE).sum())
                    y = np.clip(y, -MAX_VALUE, MAX_VALUE)
                page, slot = pool[h["tables"][r, pos // p]], pos % p
                codes = page[i * half:(i + 1) * half].reshape(nkv, p, d)
                exps = page[2 * half + i * nkv:2 * half + (i + 1) * nkv]
                if slot == 0:
                    exps[:] = 0
                for j in range(nkv):
                    was = int(exps[j])
                    n = was
                    while int(_round_shift(np.abs(y[j]).max(), n)) > 127:
                        n += 1
                    if n > was:
                        codes[j, :slot] = _round_shift(codes[j, :slot].astype(np.int64), n - was)
                        exps[j] = n
                    codes[j, slot] = _round_shift(y[j], n)
    return {"pool": pool, "q": q, "clamped": clamped, "status": np.zeros_like(h["status"])}


def _host_combine(a, b):
    m, e = (a[0] * b[0] + (1 << 30)) >> 31, a[1] + b[1] + 31
    return (m << 1, e - 1) if m < 1 << 30 else (m, e)


def _host_requant(x, scale):
    """One row of integers to codes and a scale, in Python's integers for the scale."""
    d = max(1, int(np.abs(x).max()))
    s = 31 - d.bit_length()
    dn = d << s if s >= 0 else d >> 1
    f, e, ax = 127 * (((1 << 63) + dn) // (2 * dn)), 62 - s, np.abs(x)
    low = (ax * (f & 0xfffff)) + ((np.int64(1) << (e - 1)) & 0xfffff)
    mag = ax * (f >> 20) + ((1 << (e - 1)) >> 20) + (low >> 20)
    return (np.sign(x) * np.minimum(mag >> (e - 20), 127)).astype(np.int8), _host_combine(scale, (dn, -s))


def _exact_attention(case, s):
    h, p, nh, nkv, d = _host(s), case["page"], case["heads"], case["kv_heads"], case["dim"]
    half, grp, fold = _page_bytes(case)[0], nh // nkv, h["fold"].astype(np.int64)
    codes, scales = np.zeros_like(h["codes"]), np.zeros_like(h["scales"])
    for r in range(case["rows"]):
        t0, t1 = (int(x) for x in h["row_tokens"][r:r + 2])
        width = int(h["row_start"][r]) + t1 - t0
        pages = h["pool"][h["tables"][r, :_pages_of(width, p)]]
        out = np.zeros((t1 - t0, nh, d), np.int64)
        for j in range(nkv):
            kc, vc = (pages[:, (i * nkv + j) * p * d:(i * nkv + j + 1) * p * d].reshape(-1, d)[:width].astype(np.float32) for i in (0, 1))
            ke, ve = (np.repeat(pages[:, 2 * half + i * nkv + j].astype(np.int64), p)[:width] for i in (0, 1))
            vx = vc.astype(np.float64) * (1 << ve)[:, None]
            for i in range(t1 - t0):
                w = int(h["row_start"][r]) + i + 1
                m, e = _host_combine(tuple(int(x) for x in h["q_scale"][t0 + i]), (int(h["khead_m"][j]), int(h["khead_e"][j])))
                inv = ((1 << 63) + m) // (2 * m)
                ln2, b, c = (LN2_Q * inv) >> (92 + e), (B_Q * inv) >> (92 + e), (CA_Q * inv * inv) >> (154 + 2 * e)
                q = h["q"][t0 + i].reshape(nkv, grp, d)[j].astype(np.float32)
                sc = (q @ kc[:w].T).astype(np.int64) << ke[:w]
                x = np.minimum(sc.max(1, keepdims=True) - sc, 30 * ln2)
                z = x // ln2
                ex = ((b - (x - z * ln2)) ** 2 + c) >> z
                pr = (ex * 32768) // np.maximum(ex.sum(1, keepdims=True), 1)
                out[i, j * grp:(j + 1) * grp] = (pr.astype(np.float64) @ vx[:w]).astype(np.int64)
        for i in range(t1 - t0):
            hi = (out[i] * fold[:, 1, None] + (np.int64(1) << 30)) >> 31
            codes[t0 + i], scales[t0 + i] = _host_requant(_round_shift(hi, fold[:, 2, None]).reshape(-1), SITE)
    return {"codes": codes, "scales": scales, "status": np.zeros_like(h["status"])}


def _exact_sample(case, s):
    h, v = _host(s), case["vocab"]
    tokens, mass = np.zeros_like(h["picked"]), np.zeros_like(h["mass"])
    for r in range(case["rows"]):
        ln2, b, c, top_k, top_p, min_p, random = (int(x) for x in h["rule"][r])
        legal = np.arange(v)
        if r < case["masked"]:
            legal = np.nonzero(np.unpackbits(h["mask"][r], bitorder="little")[:v])[0]
        if not len(legal):
            tokens[r] = -1
            continue
        x = h["logits"][r, legal].astype(np.int64)
        order = np.lexsort((legal, -x))
        x, legal = x[order], legal[order]
        d = x[0] - x
        w = np.where(d < 30 * ln2, ((b - d % ln2) ** 2 + c) >> np.minimum(d // ln2, 30), 0)
        if top_k:
            w = w[:top_k]
        need = -(-int(w.sum()) * top_p // 65536)
        w = w[:max(1, int(np.searchsorted(np.cumsum(w), need, "left")) + 1)]
        w = np.where(w >= -(-(b * b + c) * min_p // 65536), w, 0)
        total = int(w.sum())
        at = int(np.searchsorted(np.cumsum(w), total * random >> 32, "right"))
        tokens[r], mass[r] = legal[at], (w[at], total)
    return {"tokens": tokens, "mass": mass}


def exact(case, seed):
    if case["kind"] == "attention" and case["rows"] * case["heads"] * case["new"] * case["hi"] > 2e7:
        return None
    if case["kind"] == "store" and case["rows"] * case["new"] * case["kv_heads"] > 10000:
        return None
    return {"update": _exact_update, "compact": _exact_compact, "store": _exact_store, "attention": _exact_attention,
            "sample": _exact_sample}[case["kind"]](case, prepare(case, seed))
