"""The paged cache's operators (superslm_amd/cache_ops.py) against Python's integers and the oracle's primitives.
Integers throughout: every comparison is exact."""
import numpy as np
import pytest

import batch_ops_ref
import cache_ops_ref as ref
from cache_ops_ref import MAX_UNITS, Layout
from superslm_amd.cache_ops import CacheOps
from superslm_amd.device import Device
from superslm_amd.sslm_artifact import reciprocal_round, rope_tables, scale_me

pytestmark = pytest.mark.gpu

LEFT = 77  # what outputs hold before a call: refused rows keep it
SITE = batch_ops_ref.SITE


@pytest.fixture(scope="module")
def ops(hip_lib):
    return CacheOps(hip_lib)


@pytest.fixture(scope="module")
def dev(hip_lib):
    return Device(hip_lib)


@pytest.fixture(scope="module")
def host(oracle_lib):
    return batch_ops_ref.bind(oracle_lib)


def sync(ops):
    assert ops.lib.lib.sslm_hip_synchronize() == 0


class Batch:
    """A ragged batch over a pool of pages, in host arrays: `spans` = [(first position, new tokens)] per row."""

    def __init__(self, seed, heads, kv_heads, dim, p, spans, lead=0, tail=0, rotary=None, halves=False, spread=(0.004, 0.06), exps=(0, 8),
                 first_token=0, spare=3):
        rng = np.random.default_rng(seed)
        self.nh, self.nkv, self.d, self.p, self.spans = heads, kv_heads, dim, p, spans
        self.lay = Layout(kv_heads, dim, p, lead, tail)
        self.rows = len(spans)
        need = [-(-(s + n) // p) for s, n in spans]
        self.pages = sum(need) + spare
        order = rng.permutation(self.pages)
        self.tables = np.full((self.rows, max(need + [1]) + 1), -1, np.int32)
        at = 0
        for r, m in enumerate(need):
            self.tables[r, :m] = order[at:at + m]
            at += m
        self.pool = rng.integers(-127, 128, size=(self.pages, self.lay.page_bytes), dtype=np.int8)
        for g in range(self.pages):
            for i in range(2):
                self.lay.exps(self.pool, g, i)[:] = rng.integers(exps[0], exps[1] + 1, kv_heads)
        self.cuts = (first_token + np.cumsum([0] + [n for _, n in spans])).astype(np.int32)
        self.start = np.array([s for s, _ in spans], np.int64)
        t = self.tokens = int(self.cuts[-1]) + 2
        self.max_new, self.max_width = max([n for _, n in spans] + [1]), max([s + n for s, n in spans] + [1])
        self.rotary, self.halves = dim if rotary is None else rotary, halves
        self.cos, self.sin = rope_tables(self.max_width + 1, max(self.rotary, 2), 10000.0)
        bell = lambda *s: np.clip(np.rint(rng.standard_normal(s) * 35), -127, 127).astype(np.int8)  # noqa: E731
        self.q, self.k, self.v = bell(t, heads, dim), bell(t, kv_heads, dim), bell(t, kv_heads, dim)
        scales = lambda n, lo, hi: np.array([scale_me(float(np.exp(rng.uniform(np.log(lo), np.log(hi))))) for _ in range(n)], np.int64)  # noqa: E731
        self.k_scale, self.v_scale = scales(t, *spread), scales(t, *spread)
        unit = [scales(kv_heads, 0.9e-3, 1.4e-3) for _ in range(2)]
        self.units = [[(reciprocal_round(int(m)), int(e)) for m, e in u] for u in unit]
        # attention
        self.q_scale = scales(t, 1 / 127, 6 / 127)
        self.khead = [tuple(int(y) for y in x) for x in scales(kv_heads, 0.1 / 127 / dim ** 0.5, 0.2 / 127 / dim ** 0.5)]
        self.fold = np.zeros((heads, 3), np.int32)
        self.fold[:, 1] = rng.integers(1 << 30, 1 << 31, heads)
        self.fold[:, 2] = rng.integers(0, 6, heads)

    def common(self, dev, pool, **change):
        lay = self.lay
        self.keep = [dev.upload(self.tables), dev.upload(self.cuts), dev.upload(self.start)]
        f = dict(rows=self.rows, tokens=self.tokens, max_new=self.max_new, heads=self.nh, kv_heads=self.nkv, head_dim=self.d, pages=self.pages,
                 page_tokens=self.p, table_ld=self.tables.shape[1], pool=pool.ptr, page_bytes=lay.page_bytes, k_offset=lay.k_offset,
                 v_offset=lay.v_offset, exp_offset=lay.exp_offset, tables=self.keep[0].ptr, row_tokens=self.keep[1].ptr, row_start=self.keep[2].ptr)
        f.update(change)
        return f

    def store(self, ops, dev, stream=None, queries=True, times=1, pool=None, **change):
        """(pool, q_out, clamped, status) after the call."""
        own = pool is None
        pool = dev.upload(self.pool) if own else pool
        b = {n: dev.upload(x) for n, x in dict(
            q=self.q, k=self.k, v=self.v, ks=self.k_scale, vs=self.v_scale, cos=self.cos, sin=self.sin, rk=np.array([u[0] for u in self.units[0]], np.int64),
            ek=np.array([u[1] for u in self.units[0]], np.int64), rv=np.array([u[0] for u in self.units[1]], np.int64),
            ev=np.array([u[1] for u in self.units[1]], np.int64)).items()}
        q_out = dev.upload(np.full((self.tokens, self.nh, self.d), LEFT, np.int8))
        clamped, status = dev.upload(np.full(self.rows, LEFT, np.int32)), dev.upload(np.full(self.rows, LEFT, np.int32))
        f = self.common(dev, pool, rope_dim=self.rotary, rope_halves=int(self.halves), rope_rows=len(self.cos), rope_cos=b["cos"].ptr, rope_sin=b["sin"].ptr,
                        q=b["q"].ptr if queries else None, k=b["k"].ptr, v=b["v"].ptr, k_scale=b["ks"].ptr, v_scale=b["vs"].ptr, r_t_k=b["rk"].ptr,
                        e_t_k=b["ek"].ptr, r_t_v=b["rv"].ptr, e_t_v=b["ev"].ptr, q_out=q_out.ptr, clamped=clamped.ptr, status=status.ptr)
        f.update(change)
        call = ops.store(**f)
        for _ in range(times):
            call(stream)
        sync(ops)
        return (pool.numpy() if own else None), q_out.numpy(), clamped.numpy(), status.numpy()

    def stored(self, rows=None):
        """The same from the definition."""
        pool, q, clamped = self.pool.copy(), np.full((self.tokens, self.nh, self.d), LEFT, np.int8), np.zeros(self.rows, np.int32)
        pairs = self.rotary // 2
        for r in range(self.rows) if rows is None else rows:
            for i in range(self.spans[r][1]):
                t, pos = int(self.cuts[r]) + i, int(self.start[r]) + i
                q[t], n = ref.store_token(self.lay, pool, self.tables[r], pos, self.q[t], self.k[t], self.v[t], self.k_scale[t], self.v_scale[t],
                                          self.units, self.cos[pos, :pairs], self.sin[pos, :pairs], self.halves)
                clamped[r] += n
        return pool, q, clamped

    def attend(self, ops, dev, stream=None, **change):
        """(codes, scales, status)."""
        pool = dev.upload(self.pool)
        b = {n: dev.upload(x) for n, x in dict(q=self.q, qs=self.q_scale, km=np.array([m for m, _ in self.khead], np.int64),
                                               ke=np.array([e for _, e in self.khead], np.int64), fold=self.fold).items()}
        codes = dev.upload(np.full((self.tokens, self.nh * self.d), LEFT, np.int8))
        scales, status = dev.upload(np.full((self.tokens, 2), LEFT, np.int64)), dev.upload(np.full(self.tokens, LEFT, np.int32))
        f = self.common(dev, pool, max_width=self.max_width, q=b["q"].ptr, q_scale=b["qs"].ptr, khead_m=b["km"].ptr, khead_e=b["ke"].ptr,
                        ln2_q=batch_ops_ref.PINNED[0], b_q=batch_ops_ref.PINNED[1], ca_q=batch_ops_ref.PINNED[2], ctx_fold=b["fold"].ptr, site=SITE,
                        codes=codes.ptr, scales=scales.ptr, status=status.ptr)
        f.update(change)
        n = ops.attention_workspace(**{k: f[k] for k in ("rows", "tokens", "max_new", "heads", "kv_heads", "head_dim", "page_tokens", "max_width")})
        ws = dev.upload(np.full(n, 0xA5, np.uint8))  # whatever a workspace held before
        call = ops.attention(workspace=ws.ptr, workspace_bytes=n, **f)
        for _ in range(2):  # the second call finds the first one's workspace
            call(stream)
        sync(ops)
        return codes.numpy(), scales.numpy(), status.numpy()

    def check_attention(self, host, got, refused=None, tokens=None):
        """refused: {row: status} that its tokens have, their outputs left."""
        codes, scales, status = got
        seen = np.zeros(self.tokens, bool)
        for r, (s, n) in enumerate(self.spans):
            k, v = self.lay.values(self.pool, self.tables[r], s + n) if r not in (refused or {}) else (None, None)
            for i in range(n):
                t = int(self.cuts[r]) + i
                seen[t] = True
                if tokens is not None and t not in tokens:
                    continue
                st, c, sc = (refused[r], None, None) if r in (refused or {}) else ref.attention_token(
                    host, self.q[t], self.q_scale[t].tolist(), self.khead, k[:, :s + i + 1], v[:, :s + i + 1], self.fold)
                assert status[t] == st, (r, i, status[t], st)
                if st:
                    assert (codes[t] == LEFT).all() and (scales[t] == LEFT).all()
                else:
                    assert (codes[t] == c).all() and tuple(scales[t]) == sc, (r, i)
        assert (codes[~seen] == LEFT).all() and (scales[~seen] == LEFT).all() and (status[~seen] == LEFT).all()


# ---- landing ----
STORE = [
    # heads, kv heads, dim, page, spans, rotary, halves
    (4, 2, 32, 16, [(0, 1), (15, 1), (16, 1), (37, 1), (5, 0)], 32, False),
    (12, 2, 128, 64, [(0, 1), (63, 1), (64, 1), (777, 1)], 128, False),
    (6, 1, 64, 32, [(3, 5), (0, 33), (31, 2), (64, 64), (0, 0), (90, 7)], 64, True),
    (2, 1, 256, 16, [(7, 40), (16, 16)], 64, True),
    (7, 7, 32, 128, [(100, 60), (0, 128)], 8, False),
    (3, 3, 64, 256, [(250, 20), (0, 5)], 0, False),
    (8, 4, 128, 64, [(60, 3), (1, 62)], 72, True),
    (28, 4, 128, 16, [(8, 19)], 32, False),
    (40, 40, 32, 32, [(9, 1), (30, 2)], 32, False),
]


@pytest.mark.parametrize("case", range(len(STORE)))
def test_landing(ops, dev, case):
    nh, nkv, d, p, spans, rotary, halves = STORE[case]
    b = Batch(case, nh, nkv, d, p, spans, lead=32 * case, tail=5, rotary=rotary, halves=halves, first_token=case % 3, exps=(0, 4))
    pool, q, clamped, status = b.store(ops, dev)
    want = b.stored()
    assert (status == 0).all() and (clamped == want[2]).all()
    assert (q == want[1]).all()
    assert (pool == want[0]).all(), np.argwhere(pool != want[0])[:5]


@pytest.mark.parametrize("cuts", [[1] * 70, [7, 20, 1, 42], [69, 1], [2, 3, 64, 1], [35, 35]])
def test_every_split_of_a_span_leaves_the_same_bytes(ops, dev, cuts):
    """Pages that grow within a span, from the middle of one on."""
    whole = Batch(5, 6, 2, 64, 32, [(11, 70)], spread=(0.0005, 0.5), exps=(0, 2))
    want = whole.store(ops, dev)
    assert (want[0] == whole.stored()[0]).all()
    pool = dev.upload(whole.pool)
    q, at = np.full_like(want[1], LEFT), 0
    for n in cuts:
        whole.cuts = np.array([at, at + n], np.int32)
        whole.start, whole.max_new = np.array([11 + at], np.int64), n
        part = whole.store(ops, dev, pool=pool)
        q[at:at + n] = part[1][at:at + n]
        at += n
    assert (pool.numpy() == want[0]).all() and (q == want[1]).all()


def test_growing_pages_round_their_codes_once_more(ops, dev):
    """Tokens of very different sizes: every order of growth over one page."""
    b = Batch(8, 2, 2, 32, 64, [(20, 44), (0, 64), (63, 1), (1, 1)], spread=(1e-5, 1.0), exps=(0, 0))
    pool, _, clamped, status = b.store(ops, dev)
    want = b.stored()
    assert (pool == want[0]).all() and (clamped == want[2]).all() and clamped.sum() > 0 and (status == 0).all()


def test_clamped_values(ops, dev):
    """Landed beyond the largest unit, and turned beyond it."""
    b = Batch(9, 2, 1, 32, 16, [(0, 6), (14, 1)], spread=(0.2, 0.5))
    b.k[:, :, ::2] = 127
    b.k[:, :, 1::2] = -127
    pool, _, clamped, status = b.store(ops, dev)
    want = b.stored()
    assert (pool == want[0]).all() and (clamped == want[2]).all() and (clamped > 0).all()


@pytest.mark.parametrize("m,e", [(0, 0), (-(1 << 31), -40), ((1 << 31) - 1, 4000), (1 << 30, -5000), (1, 0), (-1500000000, -36), ((1 << 30) + 12345, -42)])
def test_scales_of_any_size(ops, dev, m, e):
    b = Batch(10, 2, 2, 32, 16, [(3, 4), (0, 1)], exps=(0, 3))
    b.k_scale[:] = (m, e)
    b.v_scale[1::2] = (m, e)
    pool, q, clamped, status = b.store(ops, dev)
    want = b.stored()
    assert (status == 0).all() and (pool == want[0]).all() and (clamped == want[2]).all()


def test_refused_rows_are_left_as_they_were(ops, dev):
    spans = [(5, 3), (0, 2), (16, 1), (30, 4), (0, 1), (2, 5), (40, 1)]
    b = Batch(11, 4, 2, 32, 16, spans)
    b.tables[0, 0] = b.pages
    b.tables[2, 1] = -1
    b.start[3] = -1
    b.start[4] = (b.tables.shape[1] * b.p)
    b.k_scale[b.cuts[5] + 3] = (1 << 31, 0)
    b.v_scale[b.cuts[6]] = (-(1 << 31) - 1, 0)
    pool, q, clamped, status = b.store(ops, dev)
    assert status.tolist() == [9, 0, 9, 9, 9, 4, 4] and (clamped == 0).all()
    want = b.stored(rows=[1])
    assert (pool == want[0]).all() and (q == want[1]).all()
    # the tables of angles end, a row has more tokens than declared, positions past 2^62
    b = Batch(12, 4, 2, 32, 16, [(5, 3), (0, 6), (20, 1), (2, 1)])
    b.start[3] = 1 << 62
    pool, q, clamped, status = b.store(ops, dev, rope_rows=20, max_new=5)
    assert status.tolist() == [0, 9, 9, 9]
    want = b.stored(rows=[0])
    assert (pool == want[0]).all() and (q == want[1]).all()


@pytest.mark.parametrize("cuts", [[0, -1, 3, 3], [3, 1, 2, 2], [0, 2, 500, 2], [-2, 1, 2, 3]])
def test_token_ranges_that_do_not_ascend(ops, dev, cuts):
    b = Batch(13, 2, 1, 32, 16, [(4, 1), (20, 1), (0, 1)])
    b.cuts = np.array(cuts, np.int32)
    b.max_new = 3
    pool, q, clamped, status = b.store(ops, dev)
    good = [r for r in range(3) if 0 <= cuts[r] <= cuts[r + 1] <= b.tokens]
    assert [s == 0 for s in status] == [r in good for r in range(3)]
    b.spans = [(int(b.start[r]), cuts[r + 1] - cuts[r]) for r in range(3)]
    want = b.stored(rows=good)
    assert (pool == want[0]).all() and (q == want[1]).all()


def test_strides_queries_in_place_and_no_queries(ops, dev):
    """q, k and v as parts of one row, as a fused projection leaves them."""
    b = Batch(14, 6, 2, 64, 32, [(3, 9), (40, 1)])
    want = b.stored()
    t, h, kv = b.tokens, b.nh * b.d, b.nkv * b.d
    fused = np.concatenate([b.q.reshape(t, h), b.k.reshape(t, kv), b.v.reshape(t, kv), np.full((t, 3), LEFT, np.int8)], 1)
    d = dev.upload(fused)
    ld = fused.shape[1]
    pool, q, _, _ = b.store(ops, dev, q=d.ptr, k=d.ptr + h, v=d.ptr + h + kv, q_ld=ld, k_ld=ld, v_ld=ld)
    assert (pool == want[0]).all() and (q == want[1]).all()
    d = dev.upload(b.q)
    pool, q, _, _ = b.store(ops, dev, q=d.ptr, q_out=d.ptr)
    got = d.numpy()
    used = slice(int(b.cuts[0]), int(b.cuts[-1]))
    assert (pool == want[0]).all() and (got[used] == want[1][used]).all() and (got[b.cuts[-1]:] == b.q[b.cuts[-1]:]).all()
    pool, q, _, _ = b.store(ops, dev, queries=False)
    assert (pool == want[0]).all() and (q == LEFT).all()


def test_two_layers_in_one_page(ops, dev):
    b = Batch(15, 4, 2, 32, 16, [(3, 20)], tail=4096)
    other = Layout(2, 32, 16, lead=b.lay.page_bytes - 2 * 2 * 16 * 32 - 16)
    first = b.store(ops, dev)[0]
    b.pool = first
    moved = b.store(ops, dev, k_offset=other.k_offset, v_offset=other.v_offset, exp_offset=other.exp_offset)[0]
    b.lay.k_offset, b.lay.v_offset, b.lay.exp_offset = other.k_offset, other.v_offset, other.exp_offset
    assert (moved == b.stored()[0]).all() and (moved != first).any()


# ---- attention ----
ATTEND = [
    # heads, kv heads, dim, page, spans
    (12, 2, 128, 64, [(0, 1), (63, 1), (64, 1), (65, 1), (99, 1)]),
    (4, 4, 32, 16, [(0, 1), (16, 1), (200, 1), (77, 1)]),
    (14, 2, 64, 32, [(500, 1), (31, 1), (1023, 1)]),
    (28, 4, 128, 64, [(2000, 1), (4095, 1), (1, 1)]),
    (8, 2, 256, 16, [(300, 1), (15, 1)]),
    (8, 2, 256, 256, [(600, 1)]),
    (20, 1, 64, 128, [(129, 1), (1000, 1)]),
    (40, 1, 32, 32, [(70, 1), (5, 1)]),
    (64, 1, 128, 64, [(200, 1)]),
    (12, 2, 128, 64, [(0, 5), (60, 9), (100, 0), (7, 1)]),
    (12, 2, 128, 32, [(40, 70), (0, 33)]),
    (6, 6, 32, 16, [(0, 130)]),
    (4, 1, 256, 128, [(300, 17), (2, 2)]),
    (16, 2, 64, 256, [(255, 40), (1, 3), (400, 1)]),
    (3, 1, 64, 16, [(10, 21), (0, 1)]),
]


@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_attention(ops, dev, host, case):
    nh, nkv, d, p, spans = ATTEND[case]
    b = Batch(100 + case, nh, nkv, d, p, spans, lead=16 * case, first_token=case % 2, exps=[(0, 8), (2, 4), (3, 3)][case % 3])
    b.check_attention(host, b.attend(ops, dev))


@pytest.mark.parametrize("scale", [1e-9, 1e-6, 3e-3, 1.0])
@pytest.mark.parametrize("spans", [[(300, 1), (40, 1)], [(90, 40)]])
def test_flat_and_peaked_scores(ops, dev, host, scale, spans):
    """Constants from where every probability is alike (sums leave the doubles) to where one position has all, and past
    the domain."""
    b = Batch(130, 8, 2, 64, 32, spans, exps=(0, 5))
    b.q_scale[:] = scale_me(scale)
    b.check_attention(host, b.attend(ops, dev))


def test_rows_of_one_batch_take_different_forms(ops, dev, host):
    b = Batch(131, 12, 2, 128, 64, [(200, 1), (90, 1), (130, 1), (3, 1), (70, 1)], exps=(1, 5))
    for r, x in enumerate((1e-9, 0.01, 1e-8, 0.02, 1.0)):
        b.q_scale[b.cuts[r]] = scale_me(x)
    b.check_attention(host, b.attend(ops, dev))
    b = Batch(132, 12, 2, 128, 64, [(200, 30)], exps=(1, 5))
    for i in range(0, 30, 4):
        b.q_scale[i] = scale_me(1e-9)
    b.check_attention(host, b.attend(ops, dev))


def test_largest_values(ops, dev, host):
    """Scores of 127 32512 256 and a context whose every value is the largest."""
    for spans in ([(100, 1)], [(50, 20)]):
        b = Batch(133, 4, 1, 256, 64, spans)
        b.pool[:] = 127
        for g in range(b.pages):
            for i in range(2):
                b.lay.exps(b.pool, g, i)[:] = 8
        b.q[:] = 127
        b.q[:, 1] = -127
        b.fold[:, 2] = 31
        b.fold[1] = (1, 0, 0)
        b.check_attention(host, b.attend(ops, dev))
        b.pool[:, :b.lay.exp_offset] = -128
        b.check_attention(host, b.attend(ops, dev))


def test_exponents_past_the_largest_count_as_it(ops, dev, host):
    for spans in ([(100, 1), (20, 1)], [(50, 20)]):
        b = Batch(134, 4, 2, 64, 16, spans)
        for g in range(0, b.pages, 2):
            b.lay.exps(b.pool, g, g // 2 % 2)[:] = 9 + g % 240
        b.check_attention(host, b.attend(ops, dev))


@pytest.mark.parametrize("chunk", [False, True])
def test_refused_rows(ops, dev, host, chunk):
    n = 5 if chunk else 1
    b = Batch(135, 12, 2, 128, 64, [(100, n), (200, n), (70, n), (10, 1), (300, n), (63, n)], exps=(2, 4))
    b.tables[0, 1] = -1
    b.tables[2, 0] = b.pages
    b.start[3] = -5
    b.start[4] = 1 << 40
    b.check_attention(host, b.attend(ops, dev), refused={0: 9, 2: 9, 3: 9, 4: 9})
    b = Batch(136, 12, 2, 128, 64, [(100, n), (200, n), (70, n)], exps=(2, 4))
    b.q_scale[b.cuts[1]] = (1 << 31, -40)
    codes, scales, status = got = b.attend(ops, dev, max_width=203 + n)
    assert status[b.cuts[1]] == 4
    b.check_attention(host, got)
    got = b.attend(ops, dev, max_width=200)  # the second row is longer than declared
    b.check_attention(host, got, refused={1: 9})


def test_chunks_longer_than_declared(ops, dev, host):
    b = Batch(137, 12, 2, 128, 64, [(10, 9), (20, 4)], exps=(2, 4))
    b.check_attention(host, b.attend(ops, dev, max_new=6), refused={0: 9})


@pytest.mark.parametrize("cuts", [[0, -1, 3, 3], [3, 1, 2, 2], [0, 2, 500, 2], [-2, 1, 2, 3]])
def test_attention_over_token_ranges_that_do_not_ascend(ops, dev, host, cuts):
    for most in (2, 3):
        b = Batch(138, 2, 1, 32, 16, [(4, 1), (20, 1), (0, 1)])
        b.cuts = np.array(cuts, np.int32)
        b.max_new = most
        good = [0 <= cuts[r] <= cuts[r + 1] <= b.tokens for r in range(3)]
        refused = {r: 9 for r in range(3) if good[r] and cuts[r + 1] - cuts[r] > most}
        b.spans = [(int(b.start[r]), cuts[r + 1] - cuts[r] if good[r] else 0) for r in range(3)]
        b.max_width = 32
        b.check_attention(host, b.attend(ops, dev), refused=refused)


def test_a_batch_does_not_change_its_rows(ops, dev):
    """A token's result is the same alone, in a batch, as a decode step or within a chunk."""
    b = Batch(139, 12, 2, 128, 32, [(333, 1), (20, 7), (900, 1), (150, 40)], exps=(1, 5))
    whole = b.attend(ops, dev)
    cuts, spans = b.cuts.copy(), b.spans
    for r, (s, n) in enumerate(spans):
        for i in (0, n - 1):
            b.rows, b.spans = 1, [(s + i, 1)]
            b.cuts, b.start = np.array([cuts[r] + i, cuts[r] + i + 1], np.int32), np.array([s + i], np.int64)
            table, b.tables = b.tables, b.tables[r:r + 1]
            b.max_new, b.max_width = 1, s + i + 1
            alone = b.attend(ops, dev)
            b.tables = table
            t = cuts[r] + i
            for x, y in zip(alone, whole):
                assert (x[t] == y[t]).all()


def test_many_rows_and_shared_pages(ops, dev, host):
    """Rows of a fork attend to the same pages."""
    b = Batch(140, 14, 2, 64, 16, [(40 + r % 30, 1) for r in range(200)], exps=(1, 4))
    for r in range(200):
        b.tables[r, :2] = b.tables[r // 10 * 10, :2]
    b.check_attention(host, b.attend(ops, dev), tokens=set(range(0, 200, 7)))


@pytest.mark.parametrize("spans", [[(9000, 1), (3, 1)], [(6000, 20)]])
def test_long_contexts(ops, dev, host, spans):
    b = Batch(141, 12, 2, 128, 64, spans, exps=(2, 4))
    b.check_attention(host, b.attend(ops, dev), tokens={0, 1, 19})


def test_landed_tokens_are_attended_to(ops, dev, host):
    """A chunk, then single tokens: what the store leaves is what the attention reads."""
    b = Batch(142, 12, 2, 128, 32, [(0, 50), (17, 1)], exps=(0, 3))
    pool, q, _, _ = b.store(ops, dev)
    b.pool = pool
    b.q[:b.cuts[-1]] = q[:b.cuts[-1]]
    b.check_attention(host, b.attend(ops, dev), tokens={0, 1, 31, 32, 49, 50})


# ---- pages ----
def change_pages(ops, dev, p, pages, tables, lengths, source, keep, room, held=None, page_bytes=64, in_place=False):
    rng = np.random.default_rng(1)
    pool = rng.integers(-127, 128, size=(pages, page_bytes), dtype=np.int8)
    b = [dev.upload(x) for x in (pool, tables, np.asarray(lengths, np.int64), np.asarray(source, np.int32), np.asarray(keep, np.int64),
                                 np.asarray(room, np.int64))]
    h = dev.upload(held) if held is not None else None
    nt = b[1] if in_place else dev.upload(np.full_like(tables, LEFT))
    nl = b[2] if in_place else dev.upload(np.full(len(tables), LEFT, np.int64))
    result = dev.upload(np.full(4, LEFT, np.int32))
    n = ops.update_workspace(len(tables), pages, tables.shape[1])
    ws = dev.upload(np.full(n, 0xA5, np.uint8))
    ops.update(rows=len(tables), pages=pages, page_tokens=p, table_ld=tables.shape[1], pool=b[0].ptr, page_bytes=page_bytes, tables=b[1].ptr,
               lengths=b[2].ptr, source=b[3].ptr, keep=b[4].ptr, room=b[5].ptr, held=h.ptr if h else None, new_tables=nt.ptr, new_lengths=nl.ptr,
               result=result.ptr, workspace=ws.ptr, workspace_bytes=n)()
    sync(ops)
    want = ref.update(tables, lengths, source, keep, room, p, pages, held)
    assert result.numpy().tolist() == want[0]
    if want[1] is None:
        assert (nt.numpy() == (tables if in_place else LEFT)).all() and (nl.numpy() == (lengths if in_place else LEFT)).all()
    else:
        assert (nt.numpy() == want[1]).all() and (nl.numpy() == room).all()
        for a, c in want[2]:
            pool[c] = pool[a]
    assert (b[0].numpy() == pool).all()
    return want


def scene(rng, rows, width, p, pages, longest):
    """Rows of which some share pages, as earlier forks leave them."""
    tables, lengths = np.full((rows, width), -1, np.int32), np.zeros(rows, np.int64)
    order, used = rng.permutation(pages), 0
    for r in range(rows):
        n = int(rng.integers(0, longest + 1))
        m = -(-n // p)
        common = 0
        if r and rng.random() < 0.6:
            o = int(rng.integers(0, r))
            common = int(rng.integers(0, min(m, -(-int(lengths[o]) // p)) + 1))
            tables[r, :common] = tables[o, :common]
        m = min(m, common + pages - used)
        tables[r, common:m] = order[used:used + m - common]
        used += m - common
        lengths[r] = min(n, m * p)
    return tables, lengths


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("rows,width,p,pages", [(1, 1, 16, 1), (4, 8, 16, 40), (7, 5, 64, 33), (30, 40, 16, 700), (150, 20, 32, 2500), (1500, 6, 16, 9000)])
def test_pages_change_hands(ops, dev, rows, width, p, pages, in_place):
    kinds = set()
    for seed in range(12 if rows < 100 else 4):
        rng = np.random.default_rng(1000 * rows + seed)
        tables, lengths = scene(rng, rows, width, p, pages, width * p)
        source = np.where(rng.random(rows) < 0.5, np.arange(rows), rng.integers(-1, rows, rows)).astype(np.int32)
        have = np.where(source >= 0, lengths[np.maximum(source, 0)], 0)
        keep = np.where(rng.random(rows) < 0.6, have, (have * rng.random(rows)).astype(np.int64))
        room = np.minimum(keep + np.where(rng.random(rows) < 0.3, 0, rng.integers(0, 3 * p if seed % 3 else 2, rows)), width * p)
        held = (rng.random(pages) < 0.1).astype(np.uint8) * 255 if seed % 2 else None
        want = change_pages(ops, dev, p, pages, tables, lengths, source, keep, room, held, in_place=in_place, page_bytes=[16, 48, 4096 + 16][seed % 3])
        kinds.add(want[0][0])
    assert 0 in kinds


def test_forks_take_pages_in_order_and_copy_the_open_one(ops, dev):
    tables = np.full((4, 6), -1, np.int32)
    tables[0, :3] = [9, 2, 5]
    want = change_pages(ops, dev, 16, 12, tables, [40, 0, 0, 0], [0, 0, 0, 0], [40] * 4, [41, 41, 50, 40], page_bytes=20 * 1024 + 32)
    # row 3 keeps the open page without writing: all others get copies
    assert want[1].tolist() == [[9, 2, 0, -1, -1, -1], [9, 2, 1, -1, -1, -1], [9, 2, 3, 4, -1, -1], [9, 2, 5, -1, -1, -1]]
    want = change_pages(ops, dev, 16, 12, tables, [40, 0, 0, 0], [0, 0, 0, 0], [40] * 4, [41, 41, 50, 41], page_bytes=33 * 1024 + 16)
    assert want[1][0].tolist() == [9, 2, 5, -1, -1, -1] and want[2] == [(5, 0), (5, 1), (5, 4)]


def test_a_pool_too_small_changes_nothing(ops, dev):
    tables = np.full((2, 4), -1, np.int32)
    tables[0, :2] = [1, 0]
    for in_place in (False, True):
        want = change_pages(ops, dev, 16, 3, tables, [32, 0], [0, 0], [32, 20], [33, 33], in_place=in_place)
        assert want[0] == [ref.EXHAUSTED, -2, 0, -1]
        want = change_pages(ops, dev, 16, 3, tables, [32, 0], [0, -1], [32, 0], [33, 0], held=np.array([0, 0, 1], np.uint8), in_place=in_place)
        assert want[0] == [ref.EXHAUSTED, -1, 0, -1]


@pytest.mark.parametrize("row,change", [(2, {"source": 5}), (1, {"source": -2}), (2, {"source": -1}), (0, {"keep": -1}), (2, {"keep": 31}), (1, {"room": 9}),
                                        (2, {"room": 65}), (1, {"length": 65}), (0, {"length": -1}), (1, {"page": 8}), (2, {"page": -1}), (0, {"keep": 1 << 62})])
def test_rows_outside_their_range_change_nothing(ops, dev, row, change):
    tables = np.full((3, 4), -1, np.int32)
    tables[:, :2] = [[0, 1], [2, 3], [4, 5]]
    lengths, source, keep, room = [30, 20, 30], [0, 1, 2], [30, 20, 30], [31, 20, 30]
    if "page" in change:
        tables[row, 1] = change["page"]
    for name, x in (("source", source), ("keep", keep), ("room", room), ("length", lengths)):
        if name in change:
            x[row] = change[name]
    assert change_pages(ops, dev, 16, 8, tables, lengths, source, keep, room)[0] == [ref.INVALID, 0, 0, row]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("rows,width,p,pages", [(1, 2, 16, 1), (3, 4, 16, 31), (5, 4, 16, 64), (40, 30, 32, 1000), (900, 8, 16, 6000), (60, 50, 16, 40000)])
def test_compaction(ops, dev, rows, width, p, pages, in_place):
    for seed in range(8 if rows < 100 else 3):
        rng = np.random.default_rng(7 * rows + seed)
        tables, lengths = scene(rng, rows, width, p, pages, width * p if seed else 0)
        held = (rng.random(pages) < [0.0, 0.2, 0.9][seed % 3]).astype(np.uint8) if seed % 4 else None
        page_bytes = [32, 4096 + 48, 16][seed % 3] if pages < 10000 else 16
        pool = rng.integers(-127, 128, size=(pages, page_bytes), dtype=np.int8)
        b = [dev.upload(x) for x in (pool, tables, lengths)]
        h = dev.upload(held) if held is not None else None
        nt = b[1] if in_place else dev.upload(np.full_like(tables, LEFT))
        m, result = dev.upload(np.full(pages, LEFT, np.int32)), dev.upload(np.full(4, LEFT, np.int32))
        n = ops.compact_workspace(rows, pages, width)
        ws = dev.upload(np.full(n, 0xA5, np.uint8))
        ops.compact(rows=rows, pages=pages, page_tokens=p, table_ld=width, pool=b[0].ptr, page_bytes=page_bytes, tables=b[1].ptr, lengths=b[2].ptr,
                    held=h.ptr if h else None, new_tables=nt.ptr, map=m.ptr, result=result.ptr, workspace=ws.ptr, workspace_bytes=n)()
        sync(ops)
        want = ref.compact(tables, lengths, p, pages, held)
        assert result.numpy().tolist() == want[0]
        assert (nt.numpy() == want[1]).all() and (m.numpy() == want[2]).all()
        for x, y in want[3]:
            pool[y] = pool[x]
        assert (b[0].numpy() == pool).all()


@pytest.mark.parametrize("length,page", [(-1, 0), (65, 0), (20, 8), (20, -1)])
def test_compaction_refuses_rows_outside_their_range(ops, dev, length, page):
    tables, lengths = np.zeros((3, 4), np.int32), np.array([16, length, 0], np.int64)
    tables[1, 1] = page
    b = [dev.upload(x) for x in (np.zeros((8, 16), np.int8), tables, lengths, np.full(8, LEFT, np.int32), np.full(4, LEFT, np.int32))]
    n = ops.compact_workspace(3, 8, 4)
    ws = dev.zeros(n, np.uint8)
    ops.compact(rows=3, pages=8, page_tokens=16, table_ld=4, pool=b[0].ptr, page_bytes=16, tables=b[1].ptr, lengths=b[2].ptr, new_tables=b[1].ptr,
                map=b[3].ptr, result=b[4].ptr, workspace=ws.ptr, workspace_bytes=n)()
    sync(ops)
    assert b[4].numpy().tolist() == [ref.INVALID, 0, 0, 1] and (b[1].numpy() == tables).all() and (b[3].numpy() == LEFT).all()


# ---- together ----
def test_a_request_that_forks(ops, dev, host):
    """One prompt, four continuations of their own for some steps, one dropped, the pool compacted, one forked again: at each
    step every row's tokens land and are attended to as in a cache of its own."""
    nh, nkv, d, p, rows, pages, width = 6, 2, 32, 16, 4, 24, 6
    rng = np.random.default_rng(3)
    model = Batch(150, nh, nkv, d, p, [(0, width * p)], exps=(0, 0))  # tables of angles for every position of a row
    lay = model.lay
    pool = dev.upload(rng.integers(-127, 128, size=(pages, lay.page_bytes), dtype=np.int8))
    tables, lengths = dev.upload(np.full((rows, width), -1, np.int32)), dev.zeros(rows, np.int64)
    result, page_map = dev.zeros(4, np.int32), dev.zeros(pages, np.int32)
    nu, nc = ops.update_workspace(rows, pages, width), ops.compact_workspace(rows, pages, width)
    ws = dev.zeros(max(nu, nc), np.uint8)
    alone = [([], []) for _ in range(rows)]  # each row's tokens (k, v, scales) as if it had a cache of its own

    def step(source, new):
        """Rows continue `source`, each with new[r] tokens."""
        have = lengths.numpy()
        keep = np.array([have[s] if s >= 0 else 0 for s in source], np.int64)
        room = keep + new
        b = [dev.upload(x) for x in (np.array(source, np.int32), keep, room)]
        ops.update(rows=rows, pages=pages, page_tokens=p, table_ld=width, pool=pool.ptr, page_bytes=lay.page_bytes, tables=tables.ptr,
                   lengths=lengths.ptr, source=b[0].ptr, keep=b[1].ptr, room=b[2].ptr, new_tables=tables.ptr, new_lengths=lengths.ptr,
                   result=result.ptr, workspace=ws.ptr, workspace_bytes=nu)()
        sync(ops)
        assert result.numpy()[0] == 0
        spans = [(int(k), int(n)) for k, n in zip(keep, new)]
        x = Batch(int(rng.integers(1 << 30)), nh, nkv, d, p, spans, exps=(0, 0), spread=(0.001, 0.2))
        x.units, x.khead, x.cos, x.sin = model.units, model.khead, model.cos, model.sin
        x.pages, x.tables = pages, tables.numpy()
        _, q, _, status = x.store(ops, dev, pool=pool)
        assert (status == 0).all()
        x.q[:x.cuts[-1]] = q[:x.cuts[-1]]
        # the same rows with pages of nobody else's
        seqs = [list(alone[s][0]) if s >= 0 else [] for s in source]
        for r in range(rows):
            for i in range(int(new[r])):
                t = int(x.cuts[r]) + i
                seqs[r].append((x.k[t], x.v[t], x.k_scale[t], x.v_scale[t]))
            alone[r] = (seqs[r], None)
        x.pool = pool.numpy()
        y = Batch(1, nh, nkv, d, p, [(0, max(1, len(s))) for s in seqs], exps=(0, 0))
        for r in range(rows):
            for i, (k, v, ks, vs) in enumerate(seqs[r]):
                ref.store_token(lay, y.pool, y.tables[r], i, x.q[0], k, v, ks, vs, model.units, model.cos[i], model.sin[i], False)
            for a, c in zip(lay.values(x.pool, x.tables[r], len(seqs[r])), lay.values(y.pool, y.tables[r], len(seqs[r]))):
                assert (a == c).all(), r
        x.check_attention(host, x.attend(ops, dev))

    step([-1] * 4, [37, 0, 0, 0])
    step([0, 0, 0, 0], [1, 2, 1, 3])
    for _ in range(3):
        step([0, 1, 2, 3], [1, 1, 1, 1])
    step([0, 3, -1, 3], [2, 1, 0, 1])
    ops.compact(rows=rows, pages=pages, page_tokens=p, table_ld=width, pool=pool.ptr, page_bytes=lay.page_bytes, tables=tables.ptr, lengths=lengths.ptr,
                new_tables=tables.ptr, map=page_map.ptr, result=result.ptr, workspace=ws.ptr, workspace_bytes=nc)()
    sync(ops)
    st, top, _, _ = result.numpy()
    used = {int(x) for r in range(rows) for x in tables.numpy()[r, :-(-int(lengths.numpy()[r]) // p)]}
    assert st == 0 and used == set(range(top))
    step([0, 1, 1, 3], [1, 1, 20, 1])
    step([0, 1, 2, 3], [1, 0, 1, 1])
