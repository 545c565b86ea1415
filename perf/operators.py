"""The operators that let one decode step serve requests that differ, in plain form and as the
framework's kernels, for timing and comparing both.

* "attention": decode attention of rows that share prompts.  A row attends to the positions
  [0, width) of its context; the first of them, the shared prompt's, lie in the prefix's KV block
  and the rest in the row's own.  Integer scores, the i-exp softmax with Q15 probabilities, P.V, the
  per-head context fold and the requant funnel over the row.
* "lora": one shared int8 projection for a batch whose rows each carry their own low-rank adapter (or
  none): GEMM, fold, adapter delta, requant funnel.
* "pick": the next token from rows of integer logits under each request's own rules: a penalty for
  tokens its context holds, biases of single tokens, a grammar's mask.  The adjusted logits and the
  lowest index of the largest.

Everything is computed in integers, so both forms give the same bits.
"""
import numpy as np
import torch

own = False

# the i-exp's constants in Q30: ln 2, and b and c / a of exp(x) ~ a ((x + b)^2 + c / a) on (-ln 2, 0]
LN2_Q, B_Q, CA_Q = (int(x * 2 ** 30) for x in (0.6931471805599453, 1.353, 0.344 / 0.3585))
SITE = (1518500250, -45)


def _attention(name, rows, heads, kv_heads, dim, prefixes, prefix, tail_lo, tail_hi, loose=0):
    c = {"kind": "attention", "rows": rows, "heads": heads, "kv_heads": kv_heads, "dim": dim, "prefixes": prefixes,
         "prefix": prefix, "own_lo": tail_lo, "own_hi": tail_hi, "loose": loose}
    return {"name": name, **c} if name else c


def _lora(name, m, n, k, adapters, rank_lo, rank_hi, bare):
    c = {"kind": "lora", "m": m, "n": n, "k": k, "adapters": adapters, "rank_lo": rank_lo, "rank_hi": rank_hi, "bare": bare}
    return {"name": name, **c} if name else c


def _pick(name, rows, vocab, history, bias, masked):
    c = {"kind": "pick", "rows": rows, "vocab": vocab, "history": history, "bias": bias, "masked": masked}
    return {"name": name, **c} if name else c


def listed():
    return [
        # two chats behind one short system prompt, a few tokens in: latency
        _attention("attn_2x96", 2, 12, 2, 128, 1, 96, 1, 9),
        # the benchmark's batch of 16 behind a prompt of 512 tokens (1.5B heads)
        _attention("attn_16x512", 16, 12, 2, 128, 1, 512, 1, 97),
        # an ordinary server: 50 requests on three prompts of odd lengths, five on none
        _attention("attn_50x1531", 50, 12, 2, 128, 3, 1531, 1, 400, loose=5),
        # long documents at the 7B heads: 96 questions about one text of 4096 tokens
        _attention("attn_96x4096", 96, 28, 4, 128, 1, 4096, 16, 384),
        # one chat turn: four rows, two adapters of rank 16 beside the o projection (1.5B)
        _lora("lora_4x1536x1536", 4, 1536, 1536, 2, 16, 16, 0),
        # the fused GEMM benchmark's projection for 32 rows with eight adapters, a quarter without one
        _lora("lora_32x4864x896", 32, 4864, 896, 8, 16, 16, 8),
        # a full decode batch, an adapter each, ranks from 8 to 64, on the deep down projection (1.5B)
        _lora("lora_64x1536x8960", 64, 1536, 8960, 64, 8, 64, 0),
        # prompts of several tenants in one chunk at the 7B depth, the entry's largest rows and columns
        _lora("lora_512x8192x3584", 512, 8192, 3584, 12, 16, 32, 100),
        # the smallest: one request over a small vocabulary
        _pick("pick_1x4096", 1, 4096, 64, 8, 0),
        # a chat batch over the full vocabulary, short histories, a few banned tokens
        _pick("pick_16x151936", 16, 151936, 200, 32, 4),
        # a large batch: long histories, many biases, half the rows under a grammar
        _pick("pick_128x151936", 128, 151936, 3000, 300, 64),
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))

    tops = {}
    for c in listed():
        w = work(c)
        tops[c["kind"]] = {k: max(w[k], tops.get(c["kind"], w)[k]) for k in w}
    while True:
        kind = rng.choice(["attention", "lora", "pick"])
        if kind == "attention":
            heads, kv, dim = rng.choice([(12, 2, 128), (12, 2, 128), (28, 4, 128), (8, 2, 128), (4, 1, 64), (4, 2, 32)])
            rows = log(1, 128)
            prefixes = rng.randrange(1, 1 + min(4, rows))
            hi = log(1, 1024)
            case = _attention(None, rows, heads, kv, dim, prefixes, log(16, 8192), rng.randrange(1, hi + 1), hi,
                              loose=rng.randrange(0, rows - prefixes + 1) if rng.random() < 0.3 else 0)
        elif kind == "lora":
            m, hi = log(1, 512), rng.choice([4, 8, 16, 16, 32, 64])
            case = _lora(None, m, 16 * log(2, 512), 16 * log(4, 640), log(1, 64), rng.randrange(1, hi + 1), hi,
                         rng.randrange(0, m) if rng.random() < 0.4 else 0)
        else:
            rows = log(1, 192)
            case = _pick(None, rows, log(500, 151936), rng.choice([0, log(1, 4096)]), rng.choice([0, log(1, 1000)]),
                         rng.randrange(0, rows + 1))
        w = work(case)
        if all(w[k] <= tops[kind][k] for k in w):
            return case


# ---- inputs ----
def _random(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _codes(g, *shape):
    return torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda", generator=g)


def _mults(g, *shape):
    return torch.randint(1 << 30, 1 << 31, shape, dtype=torch.int64, device="cuda", generator=g).to(torch.int32)


def _scales(g, n, lo, hi):
    """Carried scales (m, e), value m 2^e, spread over [lo, hi] by their logarithm."""
    value = lo * (hi / lo) ** torch.rand(n, dtype=torch.float64, device="cuda", generator=g)
    part, e = torch.frexp(value)
    return torch.stack([(part * 2.0 ** 31).to(torch.int64), e.to(torch.int64) - 31], 1)


def _groups(case):
    """The rows' prefixes: consecutive runs of rows, some longer than others, then the loose rows."""
    rows, n = case["rows"] - case["loose"], case["prefixes"]
    weights = [1 + (i * 2) % 3 for i in range(n)]
    ends = [max(i + 1, rows * sum(weights[:i + 1]) // sum(weights)) for i in range(n)]
    return [0] + ends[:-1] + [rows]


def _prefix_lengths(case):
    return [max(1, case["prefix"] - 37 * i) for i in range(case["prefixes"])]


def _own_lengths(case):
    lo, hi = case["own_lo"], case["own_hi"]
    return [lo + (i * 7919 + hi - lo) % (hi - lo + 1) for i in range(case["rows"])]


def _prepare_attention(case, seed):
    g, rows, nh, nkv, d = _random(seed), case["rows"], case["heads"], case["kv_heads"], case["dim"]
    cuts, plens, olens = _groups(case), _prefix_lengths(case), _own_lengths(case)
    which = [next((p for p in range(len(plens)) if cuts[p] <= r < cuts[p + 1]), -1) for r in range(rows)]
    widths = [olens[r] + (plens[which[r]] if which[r] >= 0 else 0) for r in range(rows)]
    cap = max(max(widths), max(plens)) + 5
    blocks = rows + len(plens)  # the rows' blocks, then the prefixes'
    pool = torch.empty((blocks, 2, nkv, cap, d), dtype=torch.int8, device="cuda")
    pool.random_(-127, 128, generator=g)
    fold = torch.zeros((nh, 3), dtype=torch.int32, device="cuda")
    fold[:, 1] = _mults(g, nh)
    fold[:, 2] = torch.randint(0, 3, (nh,), device="cuda", generator=g)
    khead = _scales(g, nkv, 0.7 / 127 / d ** 0.5, 1.5 / 127 / d ** 0.5)
    order = torch.randperm(rows, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    i32, i64 = {"dtype": torch.int32, "device": "cuda"}, {"dtype": torch.int64, "device": "cuda"}
    return {
        "case": case, "q": _codes(g, rows, nh * d), "q_scale": _scales(g, rows, 1.0 / 127, 12.0 / 127), "pool": pool,
        "khead_m": khead[:, 0].contiguous(), "khead_e": khead[:, 1].contiguous(), "fold": fold, "cap": cap,
        "block": order.cuda(), "width": torch.tensor(widths, **i64), "which": torch.tensor(which, **i64),
        "prefix_rows": torch.tensor(cuts, **i32), "prefix_block": torch.arange(rows, blocks, **i32),
        "prefix_len": torch.tensor(plens, **i64), "max_prefix": max(plens), "max_own": max(olens),
        "codes": torch.zeros((rows, nh * d), dtype=torch.int8, device="cuda"),
        "scales": torch.zeros((rows, 2), **i64), "status": torch.zeros((rows,), **i32),
    }


def _prepare_lora(case, seed):
    g, m, n, k, s = _random(seed), case["m"], case["n"], case["k"], case["adapters"]
    lo, hi = case["rank_lo"], case["rank_hi"]
    ranks = [lo + (i * 7919) % (hi - lo + 1) for i in range(s)]
    fold = torch.zeros((n, 3), dtype=torch.int32, device="cuda")
    fold[:, 1] = _mults(g, n)
    fold[:, 2] = torch.randint(4, 9, (n,), device="cuda", generator=g)
    # u comes to lie around +-40 codes; the deltas reach the size of what they are added to
    mid = int(round(np.log2(0.75 * 127 * 73 * k ** 0.5 / 40.0)))
    parts = []
    for r in ranks:
        u = torch.stack([torch.zeros(r, dtype=torch.int32, device="cuda"), _mults(g, r),
                         torch.randint(mid - 1, mid + 2, (r,), device="cuda", generator=g).to(torch.int32)], 1)
        d = torch.stack([torch.zeros(n, dtype=torch.int32, device="cuda"), _mults(g, n),
                         torch.randint(-2, 5, (n,), device="cuda", generator=g).to(torch.int32)], 1)
        parts.append((_codes(g, r, k), u, _codes(g, n, r), d))
    # an adapter's entry in the table that a program keeps on the device: four addresses and its rank
    table = torch.tensor([[x.data_ptr() for x in p] + [r] for p, r in zip(parts, ranks)], dtype=torch.int64).cuda()
    row = torch.randint(0, s, (m,), dtype=torch.int32, device="cuda", generator=g)
    row[torch.randperm(m, generator=torch.Generator().manual_seed(seed))[:case["bare"]].cuda()] = -1
    return {
        "case": case, "a": _codes(g, m, k), "w": _codes(g, n, k), "fold": fold, "in_scale": _scales(g, m, 0.005, 0.02),
        "parts": parts, "table": table, "row": row, "ranks": torch.tensor(ranks, device="cuda"),
        "codes": torch.zeros((m, n), dtype=torch.int8, device="cuda"),
        "scales": torch.zeros((m, 2), dtype=torch.int64, device="cuda"),
        "status": torch.zeros((m,), dtype=torch.int32, device="cuda"),
    }


def _prepare_pick(case, seed):
    g, rows, v = _random(seed), case["rows"], case["vocab"]
    # logits of an integer head: a bell of some 10^5 units
    logits = (torch.randn((rows, v), device="cuda", generator=g) * 120000.0).to(torch.int32)
    length = [case["history"] - (i * 7919) % (case["history"] // 2 + 1) for i in range(rows)]
    # a context repeats itself: its tokens are drawn with a heavy head, and the best ones among them
    history = (v * torch.rand((rows, max(1, case["history"])), device="cuda", generator=g) ** 3).to(torch.int32).clamp_(max=v - 1)
    history[:, ::7] = logits.argmax(1, keepdim=True).to(torch.int32)
    ids = torch.randint(0, v, (rows, max(1, case["bias"])), dtype=torch.int32, device="cuda", generator=g)
    values = torch.randint(-400000, 400001, ids.shape, dtype=torch.int32, device="cuda", generator=g)
    page = (v + 7) // 8
    mask = torch.randint(0, 256, (rows, page), dtype=torch.uint8, device="cuda", generator=g)
    mask &= torch.randint(0, 256, (rows, page), dtype=torch.uint8, device="cuda", generator=g)
    rule = torch.randint(0, 1 << 16, (rows, 3), device="cuda", generator=g)
    repetition = (65536 + rule[:, 0] // 2).to(torch.int32)  # 1.0 to 1.5 in Q16
    presence, frequency = rule[:, 1].to(torch.int32), (rule[:, 2] // 4).to(torch.int32)
    host = [x.cpu().tolist() for x in (repetition, presence, frequency)]
    table = np.zeros((rows, 7), dtype=np.int64)
    small = table.view(np.int32).reshape(rows, 14)
    for r in range(rows):
        table[r, :3] = history[r].data_ptr(), ids[r].data_ptr(), values[r].data_ptr()
        table[r, 3] = mask[r].data_ptr() if r < case["masked"] else 0
        small[r, 8:13] = length[r], case["bias"], host[0][r], host[1][r], host[2][r]
    return {
        "case": case, "logits": logits, "history": history, "length": torch.tensor(length, device="cuda"), "ids": ids,
        "values": values, "mask": mask, "repetition": repetition, "presence": presence, "frequency": frequency,
        "table": torch.from_numpy(table).cuda(), "adjusted": torch.zeros_like(logits),
        "tokens": torch.zeros((rows,), dtype=torch.int32, device="cuda"),
    }


def prepare(case, seed):
    return {"attention": _prepare_attention, "lora": _prepare_lora, "pick": _prepare_pick}[case["kind"]](case, seed)


# ---- what a pass cannot do without ----
def work(case):
    if case["kind"] == "attention":
        nh, nkv, d = case["heads"], case["kv_heads"], case["dim"]
        cuts, plens, olens = _groups(case), _prefix_lengths(case), _own_lengths(case)
        shared = sum((cuts[p + 1] - cuts[p]) * plens[p] for p in range(len(plens)))
        by = 2 * nkv * d * (sum(plens) + sum(olens)) + case["rows"] * (2 * nh * d + 60) + 12 * nh
        return {"bytes": by, "flops": 4 * nh * d * (shared + sum(olens))}
    if case["kind"] == "lora":
        m, n, k = case["m"], case["n"], case["k"]
        lo, hi = case["rank_lo"], case["rank_hi"]
        ranks = [lo + (i * 7919) % (hi - lo + 1) for i in range(case["adapters"])]
        mean = sum(ranks) / len(ranks)
        # with fewer rows than adapters, as many adapters as rows at most
        used = min(len(ranks), m - case["bare"]) * (mean * (k + n + 12) + 12 * n)
        return {"bytes": m * k + n * k + 12 * n + used + m * n + 44 * m,
                "flops": 2 * m * n * k + 2 * (m - case["bare"]) * mean * (k + n)}
    rows, v = case["rows"], case["vocab"]
    return {"bytes": 8 * rows * v + case["masked"] * ((v + 7) // 8) + rows * (3 * case["history"] + 8 * case["bias"] + 60),
            "flops": rows * v}


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


def _plain_attention(s):
    case = s["case"]
    rows, nh, nkv, d, cap = case["rows"], case["heads"], case["kv_heads"], case["dim"], s["cap"]
    grp, dev = nh // nkv, s["q"].device
    # the softmax's integer constants per (row, kv head), from the scale of one unit of score
    sm, se = _combine(s["q_scale"][:, :1], s["q_scale"][:, 1:], s["khead_m"][None], s["khead_e"][None])
    r = _reciprocal(sm)
    q_ln2, q_b = (LN2_Q * r) >> (92 + se), (B_Q * r) >> (92 + se)
    ca = CA_Q * r
    q_c = (r * (ca >> 31) + ((r * (ca & 0x7fffffff)) >> 31)) >> (123 + 2 * se)
    q_ln2, q_b, q_c = (x[:, :, None, None] for x in (q_ln2, q_b, q_c))
    q = s["q"].view(rows, nkv, grp, d).float()
    own = s["pool"][s["block"].long()]
    pre = s["pool"][s["prefix_block"].long()]
    which, plen = s["which"], s["prefix_len"]
    start = torch.where(which >= 0, plen[which.clamp(min=0)], 0)
    # the shared part: each prefix's keys against the rows of its run, padded to the longest run
    np_, mp, cuts = len(plen), s["max_prefix"], s["prefix_rows"].long()
    runs = _groups(case)
    most = max(b - a for a, b in zip(runs, runs[1:]))
    at = cuts[:-1, None] + torch.arange(most, device=dev)
    inside = at < cuts[1:, None]
    at = torch.where(inside, at, 0)
    kp, vp = (pre[:, i, :, :mp].float() for i in (0, 1))
    qs = q[at].transpose(1, 2).reshape(np_, nkv, most * grp, d)
    shared = torch.matmul(qs, kp.transpose(2, 3).contiguous()).view(np_, nkv, most, grp, mp).transpose(1, 2)
    home = torch.zeros((rows,), dtype=torch.int64, device=dev)
    home = torch.where(which >= 0, which * most + torch.arange(rows, device=dev) - cuts[which.clamp(min=0)], home)
    shared = shared.reshape(np_ * most, nkv, grp, mp)[home].to(torch.int64)
    # the rows' own part, positions [start, width)
    mo = s["max_own"]
    pos = start[:, None] + torch.arange(mo, device=dev)
    live_own = pos < s["width"][:, None]
    pos = pos.clamp(max=cap - 1)[:, None, :, None].expand(rows, nkv, mo, d)
    ko, vo = (torch.gather(own[:, i], 2, pos).float() for i in (0, 1))
    mine = torch.matmul(q, ko.transpose(2, 3).contiguous()).to(torch.int64)
    live = torch.cat([torch.arange(mp, device=dev) < start[:, None], live_own], 1)[:, None, None, :]
    score = torch.cat([shared, mine], 3)
    top = torch.where(live, score, -(1 << 40)).amax(3, keepdim=True)
    x = torch.minimum(top - score, 30 * q_ln2).clamp(min=0)
    z = x // q_ln2
    base = q_b - (x - z * q_ln2)
    e = torch.where(live, (base * base + q_c) >> z, 0)
    p = ((e << 15) // e.sum(3, keepdim=True).clamp(min=1)).float()
    # P.V: at most 32768 * 127 in all, exact in 32-bit floats
    pp = torch.zeros((np_ * most, nkv, grp, mp), device=dev)
    pp[home[which >= 0]] = p[which >= 0][..., :mp]
    pp = pp.view(np_, most, nkv, grp, mp).transpose(1, 2).reshape(np_, nkv, most * grp, mp)
    ctx = torch.matmul(pp, vp).view(np_, nkv, most, grp, d).transpose(1, 2).reshape(np_ * most, nkv, grp, d)[home]
    ctx = torch.where((which >= 0)[:, None, None, None], ctx, 0.0) + torch.matmul(p[..., mp:].contiguous(), vo)
    ctx = ctx.to(torch.int64).view(rows, nh, d)
    fold = s["fold"].to(torch.int64)
    x = _shift_away(_srdhm(ctx, fold[:, 1, None]), fold[:, 2, None]).view(rows, nh * d)
    site = torch.tensor(SITE, dtype=torch.int64, device=dev)
    codes, scales = _funnel(x, site[0].expand(rows), site[1].expand(rows))
    return {"codes": codes, "scales": scales, "status": torch.zeros((rows,), dtype=torch.int32, device=dev)}


def _plain_lora(s):
    case, dev = s["case"], s["a"].device
    m, n = case["m"], case["n"]
    a = s["a"].double()
    # sums pass 2^24: products in 64 bits
    acc = torch.matmul(a, s["w"].double().t()).to(torch.int64)
    fold = s["fold"].to(torch.int64)
    x = _shift_away(_srdhm(acc, fold[:, 1]), fold[:, 2])
    # every adapter's A against every row; a row then keeps its own adapter's part
    aa, uf = torch.cat([p[0] for p in s["parts"]]), torch.cat([p[1] for p in s["parts"]]).to(torch.int64)
    owner = torch.repeat_interleave(torch.arange(case["adapters"], device=dev), s["ranks"])
    u = torch.matmul(a, aa.double().t()).to(torch.int64)
    u = _shift_away(_srdhm(u, uf[:, 1]), uf[:, 2]).clamp(-127, 127)
    u = torch.where(owner[None] == s["row"][:, None], u, 0).float()
    d = torch.matmul(u, torch.cat([p[2] for p in s["parts"]], 1).float().t()).to(torch.int64)
    df = torch.stack([p[3] for p in s["parts"]])[s["row"].long().clamp(min=0)].to(torch.int64)
    ex = df[..., 2]
    d = _srdhm(d, df[..., 1])
    d = torch.where(ex >= 0, _shift_away(d, ex.clamp(min=0)), (d << (-ex).clamp(min=0)).clamp(-(1 << 31), (1 << 31) - 1))
    x = x + torch.where(s["row"][:, None] >= 0, d, 0)
    site = torch.tensor(SITE, dtype=torch.int64, device=dev)
    sm, se = _combine(s["in_scale"][:, 0], s["in_scale"][:, 1], site[0], site[1])
    codes, scales = _funnel(x, sm, se)
    return {"codes": codes, "scales": scales, "status": torch.zeros((m,), dtype=torch.int32, device=dev)}


def _plain_pick(s):
    case, x = s["case"], s["logits"].to(torch.int64)
    rows, v, dev = case["rows"], case["vocab"], s["logits"].device
    valid = torch.arange(s["history"].shape[1], device=dev) < s["length"][:, None]
    count = torch.zeros_like(x).scatter_add_(1, s["history"].long(), valid.to(torch.int64))
    seen, rep = count > 0, s["repetition"].to(torch.int64)[:, None]
    x = torch.where(seen, torch.where(x > 0, (x << 16) // rep, (x * rep) >> 16), x)
    if case["bias"]:
        x = x.scatter_add(1, s["ids"].long(), s["values"].to(torch.int64))
    x = x - torch.where(seen, s["presence"].to(torch.int64)[:, None] + s["frequency"].to(torch.int64)[:, None] * count, 0)
    x = x.clamp(-(1 << 31), (1 << 31) - 1)
    bits = ((s["mask"][:, :, None] >> torch.arange(8, dtype=torch.uint8, device=dev)) & 1).view(rows, -1)[:, :v].bool()
    bits = bits | (torch.arange(rows, device=dev) >= case["masked"])[:, None]
    x = torch.where(bits, x, -(1 << 31))
    # the lowest index of the largest
    at = torch.where(bits & (x == torch.where(bits, x, -(1 << 40)).amax(1, keepdim=True)), torch.arange(v, device=dev), v)
    token = at.amin(1)
    return {"tokens": torch.where(token < v, token, -1).to(torch.int32), "logits": x.to(torch.int32)}


# ---- the framework's operators ----
_LIB = []


def _ops():
    if not _LIB:
        import os

        from superslm_amd.batch_ops import BatchOps
        from superslm_amd.sslm import SslmLib

        here = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        _LIB.append(BatchOps(SslmLib(os.path.join(here, "superslm_amd", "libsslm_hip.so"))))
    return _LIB[0]


def _own_call(s):
    """The call over this state's buffers, with its workspace: made once, as a server's decode loop does."""
    case, ops = s["case"], _ops()

    def space(n):
        s["workspace"] = torch.empty((n,), dtype=torch.uint8, device="cuda")
        return {"workspace": s["workspace"].data_ptr(), "workspace_bytes": n}

    p = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if case["kind"] == "attention":
        rows, nkv, d, cap = case["rows"], case["kv_heads"], case["dim"], s["cap"]
        shape = dict(rows=rows, heads=case["heads"], kv_heads=nkv, head_dim=d, prefixes=case["prefixes"],
                     max_prefix=s["max_prefix"], max_own=s["max_own"])
        return ops.shared_attention(
            **shape, **space(ops.shared_attention_workspace(**shape)), kv_pool=p["pool"], block_bytes=2 * nkv * cap * d,
            blocks=s["pool"].shape[0], k_offset=0, v_offset=nkv * cap * d, cap=cap, q=p["q"], q_scale=p["q_scale"],
            khead_m=p["khead_m"], khead_e=p["khead_e"], ln2_q=LN2_Q, b_q=B_Q, ca_q=CA_Q, ctx_fold=p["fold"], site=SITE,
            row_block=p["block"], row_width=p["width"], prefix_rows=p["prefix_rows"], prefix_block=p["prefix_block"],
            prefix_len=p["prefix_len"], codes=p["codes"], scales=p["scales"], status=p["status"])
    if case["kind"] == "lora":
        shape = dict(m=case["m"], n=case["n"], k=case["k"])
        return ops.gemm_lora_requant(
            **shape, **space(ops.gemm_lora_workspace(**shape)), a=p["a"], w=p["w"], fold=p["fold"], in_scale=p["in_scale"],
            site=SITE, adapters=p["table"], adapter_count=case["adapters"], row_adapter=p["row"], codes=p["codes"],
            scales=p["scales"], status=p["status"])
    shape = dict(rows=case["rows"], vocab=case["vocab"])
    return ops.pick_tokens(**shape, **space(ops.pick_workspace(**shape)), logits=p["logits"], rules=p["table"],
                           tokens=p["tokens"], adjusted=p["adjusted"])


def run(state):
    if not own:
        return {"attention": _plain_attention, "lora": _plain_lora, "pick": _plain_pick}[state["case"]["kind"]](state)
    if "call" not in state:
        state["call"] = _own_call(state)
    state["call"](torch.cuda.current_stream().cuda_stream)
    if state["case"]["kind"] == "pick":
        return {"tokens": state["tokens"], "logits": state["adjusted"]}
    return {"codes": state["codes"], "scales": state["scales"], "status": state["status"]}


# ---- from the definitions, in 64-bit integers on the host ----
def _np_round_shift(x, e):
    half = np.where(e > 0, np.int64(1) << np.maximum(e - 1, 0), 0)
    return np.sign(x) * ((np.abs(x) + half) >> e)


def _np_high(x, mult):
    return (x * mult + (np.int64(1) << 30)) >> 31


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
    rows, nh, nkv, d, cap = case["rows"], case["heads"], case["kv_heads"], case["dim"], s["cap"]
    grp = nh // nkv
    h = {k: v.cpu().numpy() for k, v in s.items() if isinstance(v, torch.Tensor) and k != "pool"}
    pool = s["pool"].cpu().numpy()
    codes, scales = np.zeros((rows, nh * d), np.int8), np.zeros((rows, 2), np.int64)
    fold = h["fold"].astype(np.int64)
    for r in range(rows):
        w, p = int(h["width"][r]), int(h["which"][r])
        start = int(h["prefix_len"][p]) if p >= 0 else 0
        kv = [np.concatenate([pool[h["prefix_block"][p], i, :, :start], pool[h["block"][r], i, :, start:w]], 1)
              .astype(np.float32) if p >= 0 else pool[h["block"][r], i, :, :w].astype(np.float32) for i in (0, 1)]
        out = np.zeros((nh, d), np.int64)
        for j in range(nkv):
            m, e = _host_combine((int(h["q_scale"][r, 0]), int(h["q_scale"][r, 1])), (int(h["khead_m"][j]), int(h["khead_e"][j])))
            inv = ((1 << 63) + m) // (2 * m)
            ln2, b, c = (LN2_Q * inv) >> (92 + e), (B_Q * inv) >> (92 + e), (CA_Q * inv * inv) >> (154 + 2 * e)
            q = h["q"][r].reshape(nkv, grp, d)[j].astype(np.float32)
            sc = (q @ kv[0][j].T).astype(np.int64)
            x = np.minimum(sc.max(1, keepdims=True) - sc, 30 * ln2)
            z = x // ln2
            ex = ((b - x % ln2) ** 2 + c) >> z
            pr = (ex * 32768) // np.maximum(ex.sum(1, keepdims=True), 1)
            out[j * grp:(j + 1) * grp] = (pr.astype(np.float64) @ kv[1][j].astype(np.float64)).astype(np.int64)
        x = _np_round_shift(_np_high(out, fold[:, 1, None]), fold[:, 2, None]).reshape(-1)
        codes[r], scales[r] = _host_requant(x, SITE)
    return {"codes": codes, "scales": scales, "status": np.zeros(rows, np.int32)}


def _exact_lora(case, s):
    m, n = case["m"], case["n"]
    a, w = s["a"].cpu().numpy().astype(np.float64), s["w"].cpu().numpy().astype(np.float64)
    fold, row, ins = (s[k].cpu().numpy().astype(np.int64) for k in ("fold", "row", "in_scale"))
    x = _np_round_shift(_np_high((a @ w.T).astype(np.int64), fold[:, 1]), fold[:, 2])
    for i, (pa, pu, pb, pd) in enumerate(s["parts"]):
        at = np.nonzero(row == i)[0]
        if not len(at):
            continue
        pa, pb = (t.cpu().numpy().astype(np.float64) for t in (pa, pb))
        pu, pd = (t.cpu().numpy().astype(np.int64) for t in (pu, pd))
        u = np.clip(_np_round_shift(_np_high((a[at] @ pa.T).astype(np.int64), pu[:, 1]), pu[:, 2]), -127, 127)
        t = _np_high((u.astype(np.float64) @ pb.T).astype(np.int64), pd[:, 1])
        up = np.clip(t * (np.int64(1) << np.maximum(-pd[:, 2], 0)), -(1 << 31), (1 << 31) - 1)
        x[at] += np.where(pd[:, 2] >= 0, _np_round_shift(t, np.maximum(pd[:, 2], 0)), up)
    codes, scales = np.zeros((m, n), np.int8), np.zeros((m, 2), np.int64)
    for t in range(m):
        codes[t], scales[t] = _host_requant(x[t], _host_combine((int(ins[t, 0]), int(ins[t, 1])), SITE))
    return {"codes": codes, "scales": scales, "status": np.zeros(m, np.int32)}


def _exact_pick(case, s):
    rows, v = case["rows"], case["vocab"]
    h = {k: x.cpu().numpy() for k, x in s.items() if isinstance(x, torch.Tensor)}
    out, tokens = np.empty((rows, v), np.int32), np.empty((rows,), np.int32)
    for r in range(rows):
        x = h["logits"][r].astype(np.int64)
        ids, count = np.unique(h["history"][r, :h["length"][r]], return_counts=True)
        rep, y = int(h["repetition"][r]), x[ids]
        x[ids] = np.where(y > 0, y * 65536 // rep, (y * rep) >> 16) - int(h["presence"][r]) - int(h["frequency"][r]) * count
        if case["bias"]:
            np.add.at(x, h["ids"][r], h["values"][r].astype(np.int64))
        x = np.clip(x, -(1 << 31), (1 << 31) - 1)
        legal = np.ones(v, bool)
        if r < case["masked"]:
            legal = np.unpackbits(h["mask"][r], bitorder="little")[:v].astype(bool)
            x[~legal] = -(1 << 31)
        out[r], tokens[r] = x, np.argmax(np.where(legal, x, -(1 << 40))) if legal.any() else -1
    return {"tokens": tokens, "logits": out}


def exact(case, seed):
    return {"attention": _exact_attention, "lora": _exact_lora, "pick": _exact_pick}[case["kind"]](case, prepare(case, seed))
