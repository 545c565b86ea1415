"""The paged cache's operators and sampling where offsets pass 32 bits: pools of several GB, contexts of millions of
positions, strides of more than 2^31 logits."""
import ctypes

import numpy as np
import pytest

import batch_ops_ref
import cache_ops_ref as ref
from superslm_amd.batch_ops import BatchOps, Sampling, sampling_constants
from superslm_amd.cache_ops import CacheOps
from superslm_amd.device import Device
from test_gpu_cache_ops import LEFT, SITE, Batch, change_pages, scene

pytestmark = pytest.mark.gpu


class Large:
    """Device memory too large to come from the host."""

    def __init__(self, lib, nbytes):
        self.lib = lib.lib
        self.ptr = self.lib.sslm_hip_device_alloc(nbytes)
        assert self.ptr, "device allocation failed"

    def put(self, at, x):
        x = np.ascontiguousarray(x)
        assert self.lib.sslm_hip_copy(self.ptr + at, x.ctypes.data, x.nbytes, 0) == 0

    def get(self, at, shape, dtype):
        x = np.empty(shape, dtype)
        assert self.lib.sslm_hip_copy(x.ctypes.data, self.ptr + at, x.nbytes, 1) == 0
        return x

    def free(self):
        self.lib.sslm_hip_device_free(self.ptr)


@pytest.fixture(scope="module")
def ops(hip_lib):
    return CacheOps(hip_lib)


@pytest.fixture(scope="module")
def dev(hip_lib):
    return Device(hip_lib)


@pytest.fixture(scope="module")
def host(oracle_lib):
    return batch_ops_ref.bind(oracle_lib)


@pytest.mark.parametrize("spans", [[(100, 1), (20, 1), (70, 1)], [(100, 9), (20, 3)], [(1800, 1), (20, 1)]])
def test_pools_past_32_bits(ops, dev, host, spans):
    """Pages of 1.5 GB with the layer at the end of each: offsets within a page and between pages."""
    b = Batch(160, 12, 2, 128, 256, spans, exps=(1, 4), spare=3)
    big = 1536 << 20
    lead = big - b.lay.page_bytes
    pool = Large(ops.lib, b.pages * big)
    try:
        for p in range(b.pages):
            pool.put(p * big + lead, b.pool[p])
        lay, f = b.lay, dict(page_bytes=big, k_offset=lead + b.lay.k_offset, v_offset=lead + b.lay.v_offset, exp_offset=lead + b.lay.exp_offset)
        _, q, clamped, status = b.store(ops, dev, pool=pool, **f)
        want = b.stored()
        assert (status == 0).all() and (q == want[1]).all() and b.pages * big > 1 << 32
        for p in range(b.pages):
            assert (pool.get(p * big + lead, lay.page_bytes, np.int8) == want[0][p]).all(), p
        b.pool = want[0]
        b.q[:b.cuts[-1]] = q[:b.cuts[-1]]
        b.check_attention(host, b.attend(ops, dev, pool=pool.ptr, **f))
    finally:
        pool.free()


def test_pages_past_32_bits_change_hands(ops, dev):
    big, pages = 300 << 20, 16
    pool = Large(ops.lib, pages * big)
    try:
        rng = np.random.default_rng(1)
        edge = [rng.integers(-127, 128, 4096, dtype=np.int8) for _ in range(pages)]
        for p in range(pages):
            pool.put(p * big, edge[p])
            pool.put((p + 1) * big - 4096, edge[p][::-1])
        tables = np.full((2, 4), -1, np.int32)
        tables[0, :2] = [15, 14]
        b = [dev.upload(x) for x in (tables, np.array([20, 0], np.int64), np.zeros(2, np.int32), np.array([20, 20], np.int64), np.array([21, 21], np.int64),
                                     np.zeros(4, np.int32), np.zeros(pages, np.int32))]
        n = ops.update_workspace(2, pages, 4)
        ws = dev.zeros(max(n, ops.compact_workspace(2, pages, 4)), np.uint8)
        common = dict(rows=2, pages=pages, page_tokens=16, table_ld=4, pool=pool.ptr, page_bytes=big, tables=b[0].ptr, lengths=b[1].ptr,
                      new_tables=b[0].ptr, result=b[5].ptr, workspace=ws.ptr)
        ops.update(**common, source=b[2].ptr, keep=b[3].ptr, room=b[4].ptr, new_lengths=b[1].ptr, workspace_bytes=n)()
        assert b[5].numpy().tolist() == [0, 13, 1, -1] and b[0].numpy()[:, :2].tolist() == [[15, 14], [15, 0]]
        ops.compact(**common, map=b[6].ptr, workspace_bytes=ops.compact_workspace(2, pages, 4))()
        assert b[5].numpy().tolist() == [0, 3, 2, -1] and b[0].numpy()[:, :2].tolist() == [[2, 1], [2, 0]]
        for p, was in ((0, 14), (1, 14), (2, 15)):
            assert (pool.get(p * big, 4096, np.int8) == edge[was]).all() and (pool.get((p + 1) * big - 4096, 4096, np.int8) == edge[was][::-1]).all()
    finally:
        pool.free()


def compacted(ops, dev, p, pages, tables, lengths, pool, held=None):
    """(result, new tables, map, pool) after the call."""
    b = [dev.upload(x) for x in (pool, tables, lengths, np.full_like(tables, LEFT), np.full(pages, LEFT, np.int32), np.full(4, LEFT, np.int32))]
    h = dev.upload(held) if held is not None else None
    n = ops.compact_workspace(len(tables), pages, tables.shape[1])
    ws = dev.upload(np.full(n, 0xA5, np.uint8))
    ops.compact(rows=len(tables), pages=pages, page_tokens=p, table_ld=tables.shape[1], pool=b[0].ptr, page_bytes=pool.shape[1], tables=b[1].ptr,
                lengths=b[2].ptr, held=h.ptr if h else None, new_tables=b[3].ptr, map=b[4].ptr, result=b[5].ptr, workspace=ws.ptr, workspace_bytes=n)()
    assert ops.lib.lib.sslm_hip_synchronize() == 0
    return b[5].numpy().tolist(), b[3].numpy(), b[4].numpy(), b[0].numpy()


@pytest.mark.parametrize("seed", range(3))
def test_the_most_rows_and_pages(ops, dev, seed):
    """Plans whose bitmaps fill LDS, rows that write into one another's open pages."""
    rows, width, p, pages = 4096, 40, 16, 1 << 18
    rng = np.random.default_rng(seed)
    tables, lengths = scene(rng, rows, width, p, pages, width * p)
    lengths = np.maximum(lengths - rng.integers(0, 2, rows), 0)
    source = (rng.integers(0, rows, rows), rng.integers(0, rows, rows) // 64 * 64, np.arange(rows))[seed].astype(np.int32)
    keep = lengths[source]
    room = np.minimum(keep + rng.integers(0, 3, rows), width * p)
    held = (rng.random(pages) < 0.1).astype(np.uint8) if seed else None
    result, new, _ = change_pages(ops, dev, p, pages, tables, lengths, source, keep, room, held, page_bytes=16)
    assert result[0] == 0 and (result[2] > 1000 or seed == 2)
    pool = rng.integers(-127, 128, size=(pages, 16), dtype=np.int8)
    want = ref.compact(new, room, p, pages, held)
    got = compacted(ops, dev, p, pages, new, room, pool, held)
    assert got[0] == want[0] and (got[1] == want[1]).all() and (got[2] == want[2]).all() and want[0][2] > 1000
    for x, y in want[3]:
        pool[y] = pool[x]
    assert (got[3] == pool).all()


def test_compaction_names_the_lowest_row_out_of_range(ops, dev):
    """A page of row 3 that is none, a length of row 700 and pages of later rows, however the block's waves come to them."""
    rng = np.random.default_rng(3)
    for low, length in ((3, 700), (1100, 5), (900, None)):
        tables, lengths = rng.integers(0, 50, (1200, 30)).astype(np.int32), np.full(1200, 480, np.int64)
        tables[low, 29] = 50
        tables[low + 40:, 0] = -1
        if length is not None:
            lengths[length] = -1
        pool = np.zeros((50, 16), np.int8)
        got = compacted(ops, dev, 16, 50, tables, lengths, pool)
        assert got[0] == [ref.INVALID, 0, 0, min(low, length or low)] == ref.compact(tables, lengths, 16, 50)[0]
        assert (got[1] == LEFT).all() and (got[2] == LEFT).all()


@pytest.mark.parametrize("rows,heads,width", [(40, 16, 3_500_001), (1, 2, (1 << 24) - 5)])
def test_contexts_of_millions_of_positions(ops, dev, host, rows, heads, width):
    """Kept scores past 2^31 elements, and about the widest context: rows that are alike, each with its scores elsewhere."""
    rng = np.random.default_rng(2)
    p, d = 256, 32
    lay = ref.Layout(1, d, p)
    pool = rng.integers(-127, 128, size=(5, lay.page_bytes), dtype=np.int8)
    for g in range(5):
        lay.exps(pool, g, 0)[:], lay.exps(pool, g, 1)[:] = g % 3, 4 - g
    n = -(-width // p)
    table = rng.integers(0, 5, n).astype(np.int32)
    q = rng.integers(-127, 128, size=(1, heads, d), dtype=np.int8)
    qs, ks = (1 << 30, -36), (1 << 30, -38)  # a score's unit of 2^-14: scores to some 20
    fold = np.zeros((heads, 3), np.int32)
    fold[:, 1] = 1 << 30
    k, v = (np.concatenate([lay.codes(pool, g, i)[0].astype(np.int16) << int(lay.exps(pool, g, i)[0]) for g in table])[None, :width] for i in range(2))
    want = batch_ops_ref.attention_row(host, q[0], qs, [ks], k, v, fold)
    assert want[0] == 0 and want[1].any()
    b = {x: dev.upload(y) for x, y in dict(pool=pool, tables=np.tile(table, (rows, 1)), cuts=np.arange(rows + 1, dtype=np.int32),
                                           start=np.full(rows, width - 1, np.int64), q=np.tile(q, (rows, 1, 1)), qs=np.tile(np.array([qs], np.int64), (rows, 1)),
                                           km=np.array([ks[0]], np.int64), ke=np.array([ks[1]], np.int64), fold=fold).items()}
    codes, scales, status = dev.zeros((rows, heads * d), np.int8), dev.zeros((rows, 2), np.int64), dev.upload(np.full(rows, LEFT, np.int32))
    shape = dict(rows=rows, tokens=rows, max_new=1, heads=heads, kv_heads=1, head_dim=d, page_tokens=p, max_width=width)
    nbytes = ops.attention_workspace(**shape)
    ws = Large(ops.lib, nbytes)
    try:
        ops.attention(**shape, pages=5, table_ld=n, pool=b["pool"].ptr, page_bytes=lay.page_bytes, k_offset=lay.k_offset, v_offset=lay.v_offset,
                      exp_offset=lay.exp_offset, tables=b["tables"].ptr, row_tokens=b["cuts"].ptr, row_start=b["start"].ptr, q=b["q"].ptr, q_scale=b["qs"].ptr,
                      khead_m=b["km"].ptr, khead_e=b["ke"].ptr, ln2_q=batch_ops_ref.PINNED[0], b_q=batch_ops_ref.PINNED[1], ca_q=batch_ops_ref.PINNED[2],
                      ctx_fold=b["fold"].ptr, site=SITE, codes=codes.ptr, scales=scales.ptr, status=status.ptr, workspace=ws.ptr, workspace_bytes=nbytes)()
        assert ops.lib.lib.sslm_hip_synchronize() == 0
        assert (status.numpy() == 0).all() and (codes.numpy() == want[1]).all() and (scales.numpy() == np.array(want[2])).all()
    finally:
        ws.free()


def test_logit_rows_past_32_bits(hip_lib, dev):
    ops = BatchOps(hip_lib)
    rng = np.random.default_rng(5)
    rows, v, ld = 3, 20000, (1 << 30) + 4
    x = (rng.standard_normal((rows, v)) * 3000).astype(np.int32)
    logits = Large(hip_lib, (2 * ld + v) * 4)
    try:
        table, want = (Sampling * rows)(), []
        for r in range(rows):
            logits.put(r * ld * 4, x[r])
            c, u = sampling_constants(1000.0), int(rng.integers(0, 1 << 32))
            table[r] = Sampling(None, c["q_ln2"], c["q_b"], c["q_c"], 0, 60000, 0, u)
            want.append(ref.sample(x[r], None, c["q_ln2"], c["q_b"], c["q_c"], 0, 60000, 0, u))
        t = dev.upload(np.frombuffer(bytes(table), np.uint8))
        tokens, mass = dev.zeros(rows, np.int32), dev.zeros((rows, 2), np.int64)
        n = ops.sample_workspace(rows, v)
        ws = dev.zeros(n, np.uint8)
        ops.sample_tokens(rows=rows, vocab=v, logits=logits.ptr, logits_ld=ld, rules=t.ptr, tokens=tokens.ptr, mass=mass.ptr, workspace=ws.ptr, workspace_bytes=n)()
        assert hip_lib.lib.sslm_hip_synchronize() == 0
        assert [(int(a), *(int(y) for y in m)) for a, m in zip(tokens.numpy(), mass.numpy())] == want
    finally:
        logits.free()
