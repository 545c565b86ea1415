"""Single tokens' attention in each form that a batch's size chooses: a block with a row's scores in LDS, one with them in the
workspace, and rows cut into planes; sampling where a border is looked for over the whole row."""
import numpy as np
import pytest

import cache_ops_ref as ref
from superslm_amd.batch_ops import BatchOps
from superslm_amd.sslm_artifact import scale_me
from test_gpu_cache_ops import ATTEND, Batch, dev, host, ops  # noqa: F401  (fixtures)
from test_gpu_sample import check, random_rules, rule

pytestmark = pytest.mark.gpu

SINGLE = [i for i, c in enumerate(ATTEND) if all(n == 1 for _, n in c[4])]


@pytest.mark.parametrize("case", SINGLE)
def test_by_planes_whatever_the_rows_hold(ops, dev, host, case):  # noqa: F811
    """Declared rows of 16384 positions: planes with rows that end in the first of them."""
    nh, nkv, d, p, spans = ATTEND[case]
    b = Batch(100 + case, nh, nkv, d, p, spans, lead=16 * case, first_token=case % 2, exps=[(0, 8), (2, 4), (3, 3)][case % 3])
    b.check_attention(host, b.attend(ops, dev, max_width=16384))


PLANES = [
    # heads, kv heads, dim, page, spans: max_width (210 - rows kv_heads tiles) past 257000
    (4, 2, 32, 16, [(5000, 1), (1, 1)]),
    (9, 1, 32, 256, [(9001, 1), (2048, 1), (511, 1)]),
    (14, 2, 64, 16, [(3000, 1), (2999, 1)]),
    (17, 1, 64, 256, [(4097, 1), (255, 1)]),
    (12, 2, 128, 16, [(2100, 1), (1024, 1), (1023, 1)]),
    (5, 5, 128, 256, [(2561, 1)]),
    (40, 2, 128, 32, [(1900, 1)]),
    (8, 2, 256, 16, [(1800, 1), (700, 1)]),
    (3, 1, 256, 128, [(6000, 1), (0, 1)]),
    (31, 1, 256, 64, [(1700, 1)]),
]


@pytest.mark.parametrize("case", range(len(PLANES)))
def test_long_rows_by_planes(ops, dev, host, case):  # noqa: F811
    nh, nkv, d, p, spans = PLANES[case]
    b = Batch(300 + case, nh, nkv, d, p, spans, lead=16 * case, first_token=case % 2, exps=[(0, 8), (2, 4), (3, 3)][case % 3])
    assert b.max_width * (210 - b.rows * nkv * -(-nh // nkv // 16)) > 257000
    b.check_attention(host, b.attend(ops, dev))


@pytest.mark.parametrize("scale", [1e-9, 1e-7, 1e-5, 3e-3, 1.0])
def test_flat_and_peaked_scores_by_planes(ops, dev, host, scale):  # noqa: F811
    b = Batch(330, 8, 2, 64, 32, [(3000, 1), (40, 1), (1500, 1)], exps=(0, 5))
    b.q_scale[:] = scale_me(scale)
    b.check_attention(host, b.attend(ops, dev))
    b.q_scale[b.cuts[1]] = scale_me(0.01)
    b.check_attention(host, b.attend(ops, dev))


def test_refused_rows_by_planes(ops, dev, host):  # noqa: F811
    b = Batch(331, 12, 2, 128, 16, [(2000, 1), (1500, 1), (70, 1), (10, 1), (300, 1), (2200, 1)], exps=(2, 4))
    b.tables[0, 124] = -1
    b.tables[1, 0] = b.pages
    b.start[3] = -5
    b.start[4] = 1 << 40
    b.tables[5, 137] = 1 << 30  # the row's last page
    b.check_attention(host, b.attend(ops, dev), refused={0: 9, 1: 9, 3: 9, 4: 9, 5: 9})


# many rows, a few of them long; pages of the smallest and largest size.
KEPT = [
    # heads, kv heads, dim, page, rows, the long rows' widths
    (12, 2, 128, 64, 108, [7000, 2050, 4096, 5000]),
    (24, 1, 64, 16, 110, [9000, 4097, 1025]),
    (8, 2, 32, 256, 106, [17000, 8192, 8193]),
    (10, 2, 256, 32, 107, [6500, 1024, 513]),
]


@pytest.mark.parametrize("case", range(len(KEPT)))
def test_long_rows_among_many(ops, dev, host, case):  # noqa: F811
    nh, nkv, d, p, rows, longest = KEPT[case]
    rng = np.random.default_rng(400 + case)
    spans = [(int(x), 1) for x in rng.integers(0, 90, rows)]
    at = sorted(rng.permutation(rows)[:len(longest)])
    for r, width in zip(at, longest):
        spans[r] = (width - 1, 1)
    b = Batch(410 + case, nh, nkv, d, p, spans, exps=(0, 6))
    assert rows * nkv * -(-nh // nkv // 16) >= 210
    b.q_scale[b.cuts[at[1]]] = scale_me(1e-7)
    bad = at[2] + 1 if at[2] + 1 not in at and at[2] + 1 < rows else at[2] - 1
    b.tables[bad, 0] = b.pages
    tokens = {int(b.cuts[r]) for r in [*at, bad, 0, rows - 1]}
    got = b.attend(ops, dev)
    assert (got[2][b.cuts[0]:b.cuts[-1]] != 77).all()
    b.check_attention(host, got, refused={bad: 9}, tokens=tokens)
    # a page that is none, behind the first sixteen steps of a long row
    b.tables[at[0], (longest[0] - 1) // p] = -1
    b.check_attention(host, b.attend(ops, dev), refused={bad: 9, at[0]: 9}, tokens=tokens)


def shapes(kind, v, rng):
    """Logits whose order statistics an estimate from buckets misses."""
    at = np.arange(v)
    if kind == "quantised":
        return rng.standard_normal(v).round(1) * 100000
    if kind == "one bucket":  # all but a few within a bucket's width of one another
        x = rng.integers(0, 900, v)
        x[::v // 7] = rng.integers(-1000000, 1000000, len(x[::v // 7]))
        return x
    if kind == "one slice":  # the likely tokens side by side
        x = rng.integers(-400000, -300000, v)
        x[v // 3:v // 3 + 9000] = rng.integers(0, 30000, 9000)
        return x
    if kind == "heavy and flat":
        return np.where(at % 5000 == 17, 300000, 0) + rng.integers(0, 60000, v)
    if kind == "by index":
        return at * 3
    return -rng.exponential(60000.0, v)  # falling off


@pytest.mark.parametrize("kind", ["quantised", "one bucket", "one slice", "heavy and flat", "by index", "exponential"])
def test_sampling_where_estimates_miss(ops, dev, hip_lib, kind):  # noqa: F811
    v, rng = 70001, np.random.default_rng(20)
    x = np.clip(shapes(kind, v, rng), -(1 << 31), (1 << 31) - 1).astype(np.int32)
    some = np.packbits(rng.random(v) < 0.02, bitorder="little")
    few = np.packbits(rng.random(v) < 0.0003, bitorder="little")
    rules = [*random_rules(rng, 12, v, 45000.0), *(rule(45000.0, k, p, m, int(rng.integers(0, 1 << 32))) for k, p, m in (
        (0, 65536, 0), (20000, 65536, 0), (35000, 65000, 0), (5, 65536, 0), (0, 60000, 1), (0, 65535, 0), (v - 1, 65536, 0), (3000, 10000, 0)))]
    masks = [(None, some, few)[i % 3] for i in range(len(rules))]
    check(BatchOps(hip_lib), dev, np.tile(x, (len(rules), 1)), rules, masks)
    check(BatchOps(hip_lib), dev, np.tile(x, (len(rules), 1)), rules)
