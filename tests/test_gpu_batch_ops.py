"""The operators of a decode step whose rows are different requests (superslm_amd/batch_ops.py) against
the oracle's 64- and 128-bit arithmetic, row by row.  Integers throughout: every comparison is exact."""
import ctypes

import numpy as np
import pytest

import batch_ops_ref as ref
from batch_ops_ref import SITE
from superslm_amd.batch_ops import BatchOps, Lora, LogitRule
from superslm_amd.device import Device
from superslm_amd.sslm_artifact import scale_me

pytestmark = pytest.mark.gpu

LEFT = 77  # what outputs hold before a call: refused rows keep it


@pytest.fixture(scope="module")
def ops(hip_lib):
    return BatchOps(hip_lib)


@pytest.fixture(scope="module")
def dev(hip_lib):
    return Device(hip_lib)


@pytest.fixture(scope="module")
def host(oracle_lib):
    return ref.bind(oracle_lib)


def sync(ops):
    assert ops.lib.lib.sslm_hip_synchronize() == 0


# ---- attention over shared prompts ----
class Attention:
    """A batch in host arrays: `runs` = [(prefix length, rows)], then `loose` rows without a prefix."""

    def __init__(self, seed, heads, kv_heads, dim, runs, widths, scale=2e-5, cap=None, fold_identity=False):
        rng = np.random.default_rng(seed)
        self.nh, self.nkv, self.d, self.rows = heads, kv_heads, dim, len(widths)
        self.widths = np.array(widths, np.int64)
        self.plen = np.array([n for n, _ in runs] or [0], np.int64)
        cuts = np.cumsum([0] + [r for _, r in runs])
        self.prefixes, self.prefix_rows = len(runs), cuts.astype(np.int32)
        self.cap = cap or int(max(self.widths.max(), self.plen.max(), 1)) + 3
        self.blocks = self.rows + len(runs) + 1
        order = rng.permutation(self.blocks).astype(np.int32)
        self.row_block, self.prefix_block = order[:self.rows].copy(), order[self.rows:self.rows + max(1, len(runs))].copy()
        self.pool = rng.integers(-128, 128, size=(self.blocks, 2, kv_heads, self.cap, dim), dtype=np.int8)
        self.q = rng.integers(-127, 128, size=(self.rows, heads, dim), dtype=np.int8)
        # a unit of score is worth about `scale`
        self.khead = [scale_me(float(scale * 100 * x)) for x in rng.uniform(0.5, 1.5, kv_heads)]
        self.q_scale = np.array([scale_me(float(0.01 * x)) for x in rng.uniform(0.5, 2.0, self.rows)], np.int64)
        self.fold = np.zeros((heads, 3), np.int32)
        self.fold[:, 0] = int(fold_identity)
        self.fold[:, 1] = rng.integers(1 << 30, 1 << 31, heads)
        self.fold[:, 2] = rng.integers(0, 3, heads)
        self.max_prefix = int(self.plen.max())
        starts = [min(self.start(r), int(self.widths[r])) for r in range(self.rows)]
        self.max_own = int(max(max(w - s for w, s in zip(self.widths, starts)), 0))

    def prefix_of(self, r):
        return next((p for p in range(self.prefixes) if self.prefix_rows[p] <= r < self.prefix_rows[p + 1]), -1)

    def start(self, r):
        p = self.prefix_of(r)
        return int(self.plen[p]) if p >= 0 else 0

    def kv(self, r):
        w, p = int(self.widths[r]), self.prefix_of(r)
        s = min(self.start(r), w)
        own = self.pool[self.row_block[r]]
        if p < 0:
            return own[:, :, :w]
        return np.concatenate([self.pool[self.prefix_block[p]][:, :, :s], own[:, :, s:w]], 2)

    def expected(self, host, r):
        if self.widths[r] == 0:
            return ref.ROW_WIDTH, None, None
        k, v = self.kv(r)
        return ref.attention_row(host, self.q[r], self.q_scale[r].tolist(), self.khead, k, v, self.fold)

    def run(self, ops, dev, stream=None, **change):
        b = {n: dev.upload(x) for n, x in dict(
            pool=self.pool, q=self.q, q_scale=self.q_scale, km=np.array([m for m, _ in self.khead], np.int64),
            ke=np.array([e for _, e in self.khead], np.int64), fold=self.fold, block=self.row_block, width=self.widths,
            prow=self.prefix_rows, pblock=self.prefix_block, plen=self.plen).items()}
        h = self.nh * self.d
        codes, scales = dev.upload(np.full((self.rows, h), LEFT, np.int8)), dev.upload(np.full((self.rows, 2), LEFT, np.int64))
        status = dev.upload(np.full(self.rows, LEFT, np.int32))
        shape = dict(rows=self.rows, heads=self.nh, kv_heads=self.nkv, head_dim=self.d, prefixes=self.prefixes,
                     max_prefix=change.pop("max_prefix", self.max_prefix), max_own=change.pop("max_own", self.max_own))
        n = ops.shared_attention_workspace(**shape)
        ws = dev.upload(np.full(n, 0xA5, np.uint8))  # whatever a workspace held before
        half = self.nkv * self.cap * self.d
        fields = dict(shape, workspace=ws.ptr, workspace_bytes=n, kv_pool=b["pool"].ptr, block_bytes=2 * half,
                      blocks=self.blocks, k_offset=0, v_offset=half, cap=self.cap, q=b["q"].ptr,
                      q_scale=b["q_scale"].ptr, khead_m=b["km"].ptr, khead_e=b["ke"].ptr, ln2_q=ref.PINNED[0],
                      b_q=ref.PINNED[1], ca_q=ref.PINNED[2], ctx_fold=b["fold"].ptr, site=SITE,
                      row_block=b["block"].ptr, row_width=b["width"].ptr, prefix_rows=b["prow"].ptr,
                      prefix_block=b["pblock"].ptr, prefix_len=b["plen"].ptr, codes=codes.ptr, scales=scales.ptr,
                      status=status.ptr)
        fields.update(change)
        call = ops.shared_attention(**fields)
        for _ in range(2):  # the second call finds the first one's workspace
            call(stream)
        sync(ops)
        return codes.numpy(), scales.numpy(), status.numpy()

    def check(self, host, got, rows=None, expect=None):
        codes, scales, status = got
        for r in range(self.rows) if rows is None else rows:
            st, c, s = self.expected(host, r) if expect is None or r not in expect else (expect[r], None, None)
            assert status[r] == st, (r, status[r], st)
            if st:
                assert (codes[r] == LEFT).all() and (scales[r] == LEFT).all(), r
            else:
                assert tuple(scales[r].tolist()) == s and np.array_equal(codes[r], c), r


@pytest.mark.parametrize("heads,kv_heads,dim,runs,widths", [
    # one row, one position, no prefix; a prefix alone; a prefix longer than the row is wide
    (4, 2, 32, [], [1]),
    (4, 1, 64, [(5, 1)], [5]),
    (4, 1, 64, [(40, 3)], [40, 17, 41]),
    # lengths around the tiles' borders, rows of no width among them
    (12, 2, 128, [(63, 2), (64, 2), (65, 3)], [63, 80, 64, 129, 65, 0, 70]),
    (12, 2, 128, [(512, 5)], [513, 512, 600, 577, 1023]),
    (28, 4, 128, [(300, 4)], [301, 333, 364, 365, 1, 128, 257]),
    # an empty run, rows after the last run; one query head per KV head; more of them than a tile has rows
    (2, 2, 64, [(33, 2), (7, 0), (90, 1)], [34, 50, 91, 12, 0]),
    (20, 1, 64, [(130, 3)], [131, 150, 200, 66]),
    (40, 2, 32, [(95, 2)], [96, 97]),
    (6, 2, 256, [(70, 3)], [71, 100, 70, 31]),
    (32, 8, 256, [(150, 2)], [151, 290]),
    # more rows than one tile of rows, several tiles per prefix
    (12, 2, 128, [(200, 21), (77, 6)], [200 + i for i in range(21)] + [77 + 3 * i for i in range(6)] + [9, 300]),
])
def test_attention_matches_the_oracle(heads, kv_heads, dim, runs, widths, ops, dev, host):
    print(f"case attention {heads}/{kv_heads}x{dim} {runs} {widths}", flush=True)
    a = Attention(sum(widths) + dim, heads, kv_heads, dim, runs, widths)
    a.check(host, a.run(ops, dev))


@pytest.mark.parametrize("scale", [1e-2, 3e-4, 1e-6, 3e-7, 1.6e-7])
def test_attention_over_the_softmax_scales(scale, ops, dev, host):
    """From peaked rows (q_ln2 of a few dozen units) to flat ones whose i-exp values and sums pass 32
    and 52 bits; past them the softmax's own gate refuses the row."""
    print(f"case attention scale {scale}", flush=True)
    a = Attention(11, 12, 2, 128, [(333, 4)], [333, 350, 400, 461, 90], scale=scale)
    a.check(host, a.run(ops, dev))


def test_attention_ties_identity_fold_and_extreme_codes(ops, dev, host):
    a = Attention(5, 8, 2, 64, [(150, 3)], [151, 215, 150, 64], scale=1e-4, fold_identity=True)
    a.pool[...] = -128  # every score of a row the same
    a.q[0] = 127
    a.q[1] = -128
    print("case attention ties", flush=True)
    a.check(host, a.run(ops, dev))


def test_attention_long_prefix_and_many_splits(ops, dev, host):
    print("case attention long", flush=True)
    a = Attention(6, 4, 1, 64, [(9001, 2)], [9002, 9700, 3100])
    a.check(host, a.run(ops, dev))


def test_attention_looser_maxima_change_nothing(ops, dev, host):
    a = Attention(7, 12, 2, 128, [(100, 2), (51, 1)], [101, 130, 60, 20])
    want = a.run(ops, dev)
    a.check(host, want)
    for more in (1, 500, 5000):
        print(f"case attention maxima +{more}", flush=True)
        got = a.run(ops, dev, max_prefix=a.max_prefix + more, max_own=a.max_own + more)
        assert all(np.array_equal(x, y) for x, y in zip(got, want))


def test_attention_block_with_offsets(ops, dev, host):
    """K and V of one layer inside a larger block, V before K."""
    a = Attention(8, 4, 2, 32, [(20, 2)], [21, 30, 5])
    half = a.nkv * a.cap * a.d
    block = 16 + 2 * half + 48
    big = np.full((a.blocks, block), 99, np.int8)
    big[:, 16:16 + half] = a.pool[:, 1].reshape(a.blocks, -1)
    big[:, 16 + half:16 + 2 * half] = a.pool[:, 0].reshape(a.blocks, -1)
    d = dev.upload(big)
    print("case attention offsets", flush=True)
    a.check(host, a.run(ops, dev, kv_pool=d.ptr, block_bytes=block, k_offset=16 + half, v_offset=16))


def test_attention_refuses_rows_by_their_status(ops, dev, host):
    """Lengths and block indexes outside what the call declares, and scales outside the softmax's
    domain: the row's status says so, its outputs stay, the other rows are computed."""
    a = Attention(9, 8, 2, 64, [(40, 4), (30, 2)], [45, 44, 43, 42, 31, 33, 12, 9, 8, 7, 6])
    a.row_block[1] = a.blocks
    a.row_block[2] = -1
    a.widths[6] = a.cap + 1
    a.widths[7] = -3
    a.q_scale[8] = 1 << 31, -40
    a.q_scale[9] = 1 << 30, 300   # a scale so large that no constant of the i-exp is left
    # so small that the shift of c / a, 30 + 124 + 2 e with e = -70 + khead's (-40) + 31, is below zero
    a.q_scale[10] = 1 << 30, -70
    a.prefix_block[1] = 1000
    expect = {r: ref.POSITION_OVER_CAP for r in (1, 2, 6, 7, 4, 5)}
    print("case attention refusals", flush=True)
    got = a.run(ops, dev, max_own=12)
    assert got[2][8] == ref.SCALE_MANTISSA and got[2][9] == ref.REFUSED and got[2][10] == ref.SCALE_DERIVATION
    a.check(host, got, expect=expect)
    # maxima below the lengths
    a = Attention(9, 8, 2, 64, [(40, 2)], [45, 44, 12])
    got = a.run(ops, dev, max_prefix=39)
    a.check(host, got, expect={0: ref.POSITION_OVER_CAP, 1: ref.POSITION_OVER_CAP})
    got = a.run(ops, dev, max_own=4)
    a.check(host, got, expect={0: ref.POSITION_OVER_CAP, 2: ref.POSITION_OVER_CAP})


@pytest.mark.parametrize("runs,widths", [([(9001, 2)], [9051, 9010]), ([], [9001]), ([(20000, 1)], [29000])])
def test_attention_of_few_rows_over_many_planes(runs, widths, ops, dev, host):
    b = Attention(23, 4, 1, 32, runs, widths, scale=4e-5)
    b.check(host, b.run(ops, dev))


@pytest.mark.parametrize("runs,widths", [([(40, 2)], [45, 130, 7]), ([(1900, 3)], [1950, 2100, 1901, 800])])
def test_attention_in_a_pool_past_32_bits(runs, widths, ops, dev, host):
    """Blocks of 512 MB: heads, V and blocks lie past 2^31 and 2^32 bytes; one-launch rows and planes."""
    b = Attention(21, 12, 2, 128, runs, widths)
    cap = 1 << 20
    half = 2 * cap * 128
    alloc, copy = ops.lib.lib.sslm_hip_device_alloc, ops.lib.lib.sslm_hip_copy
    used = sorted({*b.row_block.tolist(), *b.prefix_block.tolist()})
    far = {blk: 9 - i for i, blk in enumerate(reversed(used))}  # the last blocks of ten
    pool = alloc(10 * 2 * half)
    assert pool
    try:
        for blk, at in far.items():
            for kv in range(2):
                for h in range(2):
                    rows = np.ascontiguousarray(b.pool[blk, kv, h])
                    assert copy(pool + at * 2 * half + kv * half + h * cap * 128, rows.ctypes.data, rows.nbytes, 0) == 0
        row_block, prefix_block = (dev.upload(np.array([far[x] for x in v.tolist()], np.int32)) for v in (b.row_block, b.prefix_block))
        print("case pool past 32 bits", runs, flush=True)
        b.check(host, b.run(ops, dev, kv_pool=pool, block_bytes=2 * half, v_offset=half, cap=cap, blocks=10,
                            row_block=row_block.ptr, prefix_block=prefix_block.ptr))
    finally:
        ops.lib.lib.sslm_hip_device_free(pool)


# ---- a projection with an adapter of its own per row ----
def make_adapter(rng, rank, n, k):
    mid = int(round(np.log2(max(2.0, 0.75 * 127 * 73 * k ** 0.5 / 40.0))))
    uf = np.stack([rng.random(rank) < 0.1, rng.integers(1 << 30, 1 << 31, rank), rng.integers(max(0, mid - 1), mid + 2, rank)], 1)
    df = np.stack([rng.random(n) < 0.1, rng.integers(1 << 30, 1 << 31, n), rng.integers(-3, 9, n)], 1)
    return (rng.integers(-128, 128, size=(rank, k), dtype=np.int8), np.ascontiguousarray(uf.astype(np.int32)),
            rng.integers(-128, 128, size=(n, rank), dtype=np.int8), np.ascontiguousarray(df.astype(np.int32)))


class LoraBatch:
    def __init__(self, seed, m, n, k, ranks, rows):
        rng = np.random.default_rng(seed)
        self.m, self.n, self.k = m, n, k
        self.a = rng.integers(-127, 128, size=(m, k), dtype=np.int8)
        self.w = rng.integers(-127, 128, size=(n, k), dtype=np.int8)
        self.fold = np.zeros((n, 3), np.int32)
        self.fold[:, 0] = rng.random(n) < 0.05
        self.fold[:, 1] = rng.integers(1 << 30, 1 << 31, n)
        self.fold[:, 2] = rng.integers(0, 12, n)
        self.in_scale = np.array([scale_me(float(x)) for x in rng.uniform(0.001, 0.1, m)], np.int64)
        self.adapters = [make_adapter(rng, r, n, k) for r in ranks]
        self.rows = np.array([rows[t % len(rows)] for t in range(m)], np.int32)

    def run(self, ops, dev, edit=None, **change):
        m, n, k = self.m, self.n, self.k
        b = [dev.upload(x) for x in (self.a, self.w, self.fold, self.in_scale, self.rows)]
        parts = [[dev.upload(x) for x in ad] for ad in self.adapters]
        table = (Lora * max(1, len(parts)))(*[Lora(p[0].ptr, p[1].ptr, p[2].ptr, p[3].ptr, p[0].shape[0], 0) for p in parts])
        if edit:
            edit(table)
        dt = dev.upload(np.frombuffer(bytes(table), np.uint8))
        codes, scales = dev.upload(np.full((m, n), LEFT, np.int8)), dev.upload(np.full((m, 2), LEFT, np.int64))
        status = dev.upload(np.full(m, LEFT, np.int32))
        need = ops.gemm_lora_workspace(m, n, k)
        ws = dev.upload(np.full(need, 0xA5, np.uint8))
        fields = dict(workspace=ws.ptr, workspace_bytes=need, site=SITE, m=m, n=n, k=k, adapter_count=len(parts),
                      a=b[0].ptr, w=b[1].ptr, fold=b[2].ptr, in_scale=b[3].ptr, adapters=dt.ptr, row_adapter=b[4].ptr,
                      codes=codes.ptr, scales=scales.ptr, status=status.ptr)
        fields.update(change)
        call = ops.gemm_lora_requant(**fields)
        for _ in range(2):
            call()
        sync(ops)
        return codes.numpy(), scales.numpy(), status.numpy()

    def check(self, host, got, refused=()):
        codes, scales, status = got
        for t in range(self.m):
            if t in refused:
                assert status[t] == -1 and (codes[t] == LEFT).all() and (scales[t] == LEFT).all(), t
                continue
            i = self.rows[t]
            st, c, s = ref.lora_row(host, self.a[t], self.in_scale[t].tolist(), self.w, self.fold,
                                    self.adapters[i] if i >= 0 else None)
            assert status[t] == st, (t, status[t], st)
            if st:
                assert (codes[t] == LEFT).all() and (scales[t] == LEFT).all(), t
            else:
                assert tuple(scales[t].tolist()) == s and np.array_equal(codes[t], c), t


@pytest.mark.parametrize("m,n,k,ranks,rows", [
    (1, 16, 16, [1], [0]),
    (1, 1536, 1536, [16], [0]),
    (3, 48, 80, [1, 2, 3], [2, 0, 1]),
    (4, 1536, 1536, [16, 16], [0, 1, -1, 0]),
    (5, 320, 896, [7, 64, 33, 4], [1, 3, 0, 2]),
    (16, 512, 1552, [16] * 16, list(range(16))),
    (33, 4864, 896, [8, 12, 20, 5], [0, -1, 1, 2, 3, -5]),
    (64, 1536, 8960, [64, 32, 16], [0, 1, 2, -1]),
    (65, 128, 256, [16, 31], [1, 0]),
    (130, 400, 176, [6], [-1, 0]),
    (200, 640, 1536, [16, 24], [0, -1, 1]),
    (512, 256, 384, [3, 48], [1, 0, 0]),
    (7, 8192, 64, [16], [0, -1]),
    (9, 64, 20480, [16, 64], [1, 0]),
])
def test_lora_matches_the_oracle(m, n, k, ranks, rows, ops, dev, host):
    print(f"case lora {m}x{n}x{k} {ranks}", flush=True)
    b = LoraBatch(m + n + k, m, n, k, ranks, rows)
    b.check(host, b.run(ops, dev))


@pytest.mark.parametrize("n,lo,hi", [(32, -31, 32), (2064, -31, 32), (2064, -3, 5), (2064, 5, 32)])
def test_lora_every_rank_and_exponent(n, lo, hi, ops, dev, host):
    """One row per rank, its B rows beginning at every byte of their words; delta exponents over the whole
    range, with deltas that saturate and that meet ties, and over parts of it, so that no delta hides the
    others; folds with hardly a shift, so that sums are large."""
    b = LoraBatch(n, 64, n, 256, list(range(1, 65)), list(range(64)))
    rng = np.random.default_rng(n + 1)
    for a, uf, lb, df in b.adapters:
        uf[:, 2] = rng.integers(8, 20, len(uf))
        df[:, 2] = rng.integers(lo, hi, n)
        df[::7, 1] = -(1 << 31)
        df[::5, 1] = 1 << 30
    b.fold[:, 2] = rng.integers(0, 2, n)
    b.check(host, b.run(ops, dev))



def test_lora_without_adapters_is_the_shared_projection(ops, dev, host):
    b = LoraBatch(3, 6, 96, 128, [], [-1])
    print("case lora none", flush=True)
    b.check(host, b.run(ops, dev, adapters=None))


def test_lora_refuses_rows_by_their_status(ops, dev, host):
    b = LoraBatch(4, 8, 64, 64, [4, 8, 5], [0, 1, 2, 3, -1, 1, 2, 0])

    def edit(table):
        table[2].rank = 65

    print("case lora refusals", flush=True)
    b.check(host, b.run(ops, dev, edit=edit), refused=(2, 3, 6))
    b = LoraBatch(5, 3, 64, 64, [4], [0])
    b.in_scale[1] = 1 << 31, -40  # outside the mantissa's domain
    got = b.run(ops, dev)
    assert got[2][1] == ref.SCALE_MANTISSA
    b.check(host, got)


@pytest.mark.parametrize("field", ["a", "ufold", "b", "dfold", "misaligned"])
def test_lora_refuses_pointers_by_the_row(field, ops, dev, host):
    b = LoraBatch(6, 4, 64, 64, [4, 8], [0, 1, -1, 1])

    def edit(table):
        if field == "misaligned":
            table[1].a += 8
        else:
            setattr(table[1], field, None)

    print("case lora pointers", field, flush=True)
    b.check(host, b.run(ops, dev, edit=edit), refused=(1, 3))


# ---- the next token under each row's rules ----
class Pick:
    def __init__(self, seed, vocab, rows):
        """rows: dicts with history, bias (pairs), mask (legal ids or None), repetition, presence, frequency."""
        rng = np.random.default_rng(seed)
        self.vocab, self.rules = vocab, rows
        self.logits = (rng.standard_normal((len(rows), vocab)) * 1e5).astype(np.int32)

    def mask(self, r):
        legal = self.rules[r].get("mask")
        if legal is None:
            return None
        m = np.zeros((self.vocab + 7) // 8, np.uint8)
        for j in legal:
            m[j >> 3] |= 1 << (j & 7)
        return m

    def run(self, ops, dev, ld=None, adjusted_ld=None, in_place=False, no_adjusted=False, edit=None):
        rows, v = len(self.rules), self.vocab
        ld, ald = ld or v, adjusted_ld or v
        wide = np.full((rows, ld), 2 ** 31 - 1, np.int32)
        wide[:, :v] = self.logits
        d = dev.upload(wide)
        out = d if in_place else dev.upload(np.full((rows, ald), LEFT, np.int32))
        keep, table = [], (LogitRule * rows)()
        for r, u in enumerate(self.rules):
            h = np.array(u.get("history", []), np.int32)
            ids = np.array([i for i, _ in u.get("bias", [])], np.int32)
            vals = np.array([b for _, b in u.get("bias", [])], np.int64).astype(np.int32)
            m = self.mask(r)
            up = [dev.upload(x) if x is not None and len(x) else None for x in (h, ids, vals, m)]
            keep.append(up)
            table[r] = LogitRule(*[x.ptr if x else None for x in up], len(h), len(ids), u.get("repetition", 65536),
                                 u.get("presence", 0), u.get("frequency", 0), 0)
        if edit:
            edit(table)
        dt = dev.upload(np.frombuffer(bytes(table), np.uint8))
        tokens = dev.upload(np.full(rows, LEFT, np.int32))
        need = ops.pick_workspace(rows, v)
        ws = dev.upload(np.full(need, 0xA5, np.uint8))
        call = ops.pick_tokens(workspace=ws.ptr, workspace_bytes=need, rows=rows, vocab=v, logits=d.ptr, logits_ld=ld,
                               rules=dt.ptr, tokens=tokens.ptr, adjusted=None if no_adjusted else out.ptr,
                               adjusted_ld=ld if in_place else ald)
        for _ in range(1 if in_place else 2):
            call()
        sync(ops)
        return tokens.numpy(), out.numpy(), d.numpy()

    def check(self, got, refused=()):
        tokens, out, _ = got
        for r, u in enumerate(self.rules):
            if r in refused:
                assert tokens[r] == -2 and (out[r] == LEFT).all(), r
                continue
            tok, x = ref.pick_row(self.logits[r], np.array(u.get("history", []), np.int64), u.get("bias", []), self.mask(r),
                                  u.get("repetition", 65536), u.get("presence", 0), u.get("frequency", 0))
            assert tokens[r] == tok, (r, tokens[r], tok)
            assert np.array_equal(out[r, :self.vocab], x), r
            assert (out[r, self.vocab:] == (2 ** 31 - 1 if out.shape[1] > self.vocab and out[r, -1] != LEFT else LEFT)).all()


def test_pick_rows_past_32_bits(ops, dev):
    """A row stride of 2^30 logits: the third row begins 8 GB in."""
    p = Pick(31, 5000, [dict(history=[3, 4999], presence=7), dict(), dict(history=[17] * 5, frequency=90000, mask=range(0, 5000, 3))])
    ld, alloc, copy = 1 << 30, ops.lib.lib.sslm_hip_device_alloc, ops.lib.lib.sslm_hip_copy
    logits = alloc((2 * ld + p.vocab) * 4)
    assert logits
    try:
        for r in range(3):
            row = np.ascontiguousarray(p.logits[r])
            assert copy(logits + r * ld * 4, row.ctypes.data, row.nbytes, 0) == 0
        hist = [dev.upload(np.array(u.get("history", [0]), np.int32)) for u in p.rules]
        mask = dev.upload(p.mask(2))
        table = (LogitRule * 3)(*[LogitRule(h.ptr, None, None, mask.ptr if r == 2 else None, len(u.get("history", [])), 0, 65536,
                                            u.get("presence", 0), u.get("frequency", 0), 0)
                                  for r, (h, u) in enumerate(zip(hist, p.rules))])
        dt, tokens = dev.upload(np.frombuffer(bytes(table), np.uint8)), dev.upload(np.full(3, LEFT, np.int32))
        need = ops.pick_workspace(3, p.vocab)
        ws = dev.upload(np.zeros(need, np.uint8))
        print("case rows past 32 bits", flush=True)
        ops.pick_tokens(workspace=ws.ptr, workspace_bytes=need, rows=3, vocab=p.vocab, logits=logits, logits_ld=ld, rules=dt.ptr,
                        tokens=tokens.ptr, adjusted=logits, adjusted_ld=ld)()
        sync(ops)
        for r, u in enumerate(p.rules):
            tok, x = ref.pick_row(p.logits[r], np.array(u.get("history", []), np.int64), [], p.mask(r), 65536,
                                  u.get("presence", 0), u.get("frequency", 0))
            out = np.empty(p.vocab, np.int32)
            assert copy(out.ctypes.data, logits + r * ld * 4, out.nbytes, 1) == 0
            assert tokens.numpy()[r] == tok and np.array_equal(out, x), r
    finally:
        ops.lib.lib.sslm_hip_device_free(logits)


def some_rules(seed, vocab, rows):
    rng = np.random.default_rng(seed)
    out = []
    for r in range(rows):
        n = int(rng.integers(0, 3 * vocab // 2 + 2)) if vocab < 3000 else int(rng.integers(0, 2500))
        u = {"history": (vocab * rng.random(n) ** 2).astype(int).tolist(), "repetition": int(rng.integers(30000, 120000)),
             "presence": int(rng.integers(-20000, 60000)), "frequency": int(rng.integers(-3000, 9000))}
        if r % 3 != 1:
            u["bias"] = [(int(rng.integers(0, vocab)), int(rng.integers(-300000, 300000))) for _ in range(r * 5)]
        if r % 2:
            u["mask"] = np.nonzero(rng.random(vocab) < 0.3)[0].tolist()
        out.append(u)
    return out


@pytest.mark.parametrize("vocab,rows", [(1, 2), (7, 5), (500, 6), (4095, 4), (4096, 3), (4097, 5), (9001, 4), (151936, 3)])
def test_pick_matches_the_definition(vocab, rows, ops, dev):
    print(f"case pick {vocab} x {rows}", flush=True)
    p = Pick(vocab + rows, vocab, some_rules(vocab, vocab, rows))
    p.check(p.run(ops, dev))


def test_pick_edges(ops, dev):
    """Ids outside the vocabulary, an id biased several times, one token seen thousands of times, values
    that saturate, ties (the lowest index), masks of one token, of none, and a legal INT32_MIN."""
    v, big = 5003, 2 ** 31 - 1
    p = Pick(1, v, [
        {"history": [-1, v, big, 3, 3], "frequency": 100, "repetition": 98304},
        {"bias": [(9, big), (9, big), (9, -big), (10, -big), (10, -big), (11, -5), (-4, 7), (v, 8)]},
        {"history": [17] * 9000, "frequency": big, "presence": big, "repetition": 1},
        {"mask": [4999]},
        {"mask": []},
        {"mask": [5, 6], "bias": [(5, -big), (5, -big), (6, -big), (6, -big)]},
        {},
        {"history": list(range(v)), "repetition": big, "presence": -big, "frequency": -big},
    ])
    p.logits[6] = 42
    p.logits[2, 17] = big
    p.logits[0, 3] = -(2 ** 31)
    print("case pick edges", flush=True)
    got = p.run(ops, dev)
    p.check(got)
    assert got[0][4] == -1 and got[0][5] == 5 and got[0][6] == 0


@pytest.mark.parametrize("ld,adjusted_ld", [(5000, 4800), (4801, 4803), (4804, 4801)])
def test_pick_strides_and_in_place(ld, adjusted_ld, ops, dev):
    p = Pick(ld, 4800, some_rules(3, 4800, 5))
    print(f"case pick strides {ld} {adjusted_ld}", flush=True)
    got = p.run(ops, dev, ld=ld, adjusted_ld=adjusted_ld)
    p.check(got)
    assert np.array_equal(got[2][:, :4800], p.logits)  # the input is not written
    p.check(p.run(ops, dev, ld=ld, in_place=True))
    tokens, out, _ = p.run(ops, dev, ld=ld, no_adjusted=True)
    assert (tokens == got[0]).all() and (out == LEFT).all()


def test_pick_refuses_rules_by_their_token(ops, dev):
    p = Pick(2, 600, some_rules(5, 600, 6))

    def edit(table):
        table[0].repetition_q16 = 0
        table[1].history_len = -1
        table[2].bias_count = -7
        table[3].history, table[3].history_len = None, 4

    print("case pick refusals", flush=True)
    p.check(p.run(ops, dev, edit=edit), refused=(0, 1, 2, 3))
