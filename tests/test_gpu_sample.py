"""Sampling (sslm_hip_sample_tokens) against Python's integers, row by row: every comparison is exact."""
import ctypes

import numpy as np
import pytest

import cache_ops_ref as ref
from superslm_amd.batch_ops import BatchOps, LogitRule, Sampling, sampling_constants
from superslm_amd.device import Device

pytestmark = pytest.mark.gpu

LEFT = 77


@pytest.fixture(scope="module")
def ops(hip_lib):
    return BatchOps(hip_lib)


@pytest.fixture(scope="module")
def dev(hip_lib):
    return Device(hip_lib)


def rule(unit=1000.0, top_k=0, top_p=65536, min_p=0, random=0, **change):
    return dict(sampling_constants(unit), top_k=top_k, top_p=top_p, min_p=min_p, random=random, **change)


def run(ops, dev, logits, rules, masks=None, ld=None, stream=None, mass=True):
    """logits [rows, vocab]; rules: dicts; masks: pages or None per row."""
    rows, v = logits.shape
    ld = ld or v
    host = np.full((rows, ld), -5, np.int32)
    host[:, :v] = logits
    pages = [dev.upload(m) if m is not None else None for m in (masks or [None] * rows)]
    table = (Sampling * rows)()
    for r, x in enumerate(rules):
        table[r] = Sampling(pages[r].ptr if pages[r] else None, x["q_ln2"], x["q_b"], x["q_c"], x["top_k"], x["top_p"], x["min_p"], x["random"])
    d = dev.upload(host)
    t = dev.upload(np.frombuffer(bytes(table), np.uint8))
    tokens, ms = dev.upload(np.full(rows, LEFT, np.int32)), dev.upload(np.full((rows, 2), LEFT, np.int64))
    n = ops.sample_workspace(rows, v)
    ws = dev.upload(np.full(n, 0xA5, np.uint8))
    call = ops.sample_tokens(rows=rows, vocab=v, logits=d.ptr, logits_ld=ld, rules=t.ptr, tokens=tokens.ptr,
                             mass=ms.ptr if mass else None, workspace=ws.ptr, workspace_bytes=n)
    for _ in range(2):
        call(stream)
    assert ops.lib.lib.sslm_hip_synchronize() == 0
    return tokens.numpy(), ms.numpy()


def check(ops, dev, logits, rules, masks=None, **more):
    tokens, mass = run(ops, dev, logits, rules, masks, **more)
    for r, x in enumerate(rules):
        want = ref.sample(logits[r], masks[r] if masks else None, *[x[k] for k in ("q_ln2", "q_b", "q_c", "top_k", "top_p", "min_p", "random")])
        assert (tokens[r], *mass[r]) == want, (r, x, tokens[r], mass[r], want)


def random_rules(rng, rows, vocab, unit):
    out = []
    for r in range(rows):
        form = r % 6
        top_k = [0, 1, int(rng.integers(2, 70)), 0, int(rng.integers(1, 2 * vocab)), 1 << 30][form]
        top_p = [int(rng.integers(1, 65536)), 65536, int(rng.integers(30000, 65536)), 65536, int(rng.integers(0, 65537)), 65536][form]
        min_p = [0, 0, int(rng.integers(0, 9000)), int(rng.integers(0, 3000)), int(rng.integers(0, 65537)), 0][form]
        out.append(rule(unit * float(rng.uniform(0.4, 2.0)), top_k, top_p, min_p, int(rng.integers(0, 1 << 32))))
    return out


@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 500, 4095, 4096, 4097, 8193, 32003])
def test_all_forms_of_rules(ops, dev, vocab):
    rng = np.random.default_rng(vocab)
    rows = 24
    logits = (rng.standard_normal((rows, vocab)) * 3000).astype(np.int32)
    masks = [None if r % 3 else rng.integers(0, 256, (vocab + 7) // 8, dtype=np.uint8) for r in range(rows)]
    check(ops, dev, logits, random_rules(rng, rows, vocab, 1000.0), masks)


@pytest.mark.parametrize("rows,vocab,spread", [(1, 151936, 120000), (5, 151936, 300000), (3, 262144, 20000)])
def test_full_vocabularies(ops, dev, rows, vocab, spread):
    rng = np.random.default_rng(rows)
    logits = (rng.standard_normal((rows, vocab)) * spread).astype(np.int32)
    check(ops, dev, logits, random_rules(rng, rows, vocab, 45000.0)[:rows])
    check(ops, dev, logits, [rule(45000.0, random=int(x)) for x in rng.integers(0, 1 << 32, rows)])
    check(ops, dev, logits, [rule(45000.0, top_p=60000, random=int(x)) for x in rng.integers(0, 1 << 32, rows)])


@pytest.mark.parametrize("logits", ["equal", "two", "steps", "extremes", "falling", "rising"])
def test_ties_and_extremes(ops, dev, logits):
    """Equal logits go by their index; the range of int32 from end to end."""
    v = 9000
    x = {"equal": np.full(v, 12345), "two": np.where(np.arange(v) % 5 == 0, 700, 0), "steps": np.arange(v) // 100 * 300,
         "extremes": np.where(np.arange(v) % 2 == 0, -(1 << 31), (1 << 31) - 1), "falling": -np.arange(v) * 5,
         "rising": np.arange(v) * 5}[logits].astype(np.int32)
    rng = np.random.default_rng(4)
    rules = [rule(1000.0, k, p, m, int(u)) for k, p, m in ((0, 65536, 0), (1, 65536, 0), (777, 65536, 0), (4500, 65536, 0), (0, 30000, 0), (0, 1, 0),
                                                           (0, 0, 0), (900, 40000, 100), (v, 65535, 65536), (v + 1, 65536, 1), (8999, 65535, 0))
             for u in (0, (1 << 32) - 1, rng.integers(0, 1 << 32))]
    check(ops, dev, np.tile(x, (len(rules), 1)), rules)


def test_random_numbers_at_the_borders(ops, dev):
    """Running sums that a random number falls on exactly: three tokens of weights 4, 2 and 2 (q_ln2 = 2, q_b = 2, q_c = 0)."""
    x = np.array([[0, 10, 8, 8, -50]], np.int32)
    base = dict(q_ln2=2, q_b=2, q_c=0, top_k=0, top_p=65536, min_p=0)
    rules = [dict(base, random=u) for u in (0, 1, (1 << 31) - 1, 1 << 31, (1 << 31) + 1, (1 << 30) * 3, (1 << 32) - 1, 2863311530, 2863311531)]
    check(ops, dev, np.tile(x, (len(rules), 1)), rules)


def test_rows_without_a_legal_token_and_rules_outside_their_domain(ops, dev):
    v = 5000
    rng = np.random.default_rng(9)
    good = rule(1000.0, random=5)
    bad = [dict(good, **c) for c in (dict(q_ln2=0), dict(q_ln2=-3), dict(q_b=-1), dict(q_c=-1), dict(q_b=1 << 24), dict(q_ln2=2 * good["q_b"] + 2),
                                     dict(q_c=(1 << 47) + 1), dict(q_b=0, q_c=0, q_ln2=1), dict(top_k=-1), dict(top_p=-1), dict(top_p=65537),
                                     dict(min_p=-1), dict(min_p=65537), dict(q_b=1 << 62, q_ln2=1))]
    rules = [good, *bad, good, dict(good, q_b=0, q_c=1, q_ln2=1), dict(good, q_b=11863283, q_c=0, q_ln2=2 * 11863283 + 1)]
    logits = (rng.standard_normal((len(rules), v)) * 3000).astype(np.int32)
    masks = [None] * len(rules)
    masks[0] = np.zeros((v + 7) // 8, np.uint8)
    one = np.zeros((v + 7) // 8, np.uint8)
    one[-1] = 0x80  # the vocabulary's last token alone
    masks[len(bad) + 1] = one
    check(ops, dev, logits, rules, masks)
    tokens, mass = run(ops, dev, logits, rules, masks)
    assert tokens[0] == -1 and tokens[len(bad) + 1] == v - 1 and (tokens[1:len(bad) + 1] == -2).all() and not mass[:len(bad) + 1].any()


def test_the_bits_past_the_vocabulary_are_not_read_as_tokens(ops, dev):
    v = 4099
    x = np.zeros((2, v), np.int32)
    masks = [np.full((v + 7) // 8, 255, np.uint8) for _ in range(2)]
    check(ops, dev, x, [rule(10.0, random=(1 << 32) - 1), rule(10.0, top_p=65535, random=(1 << 32) - 1)], masks)


@pytest.mark.parametrize("ld", [5001, 5003, 8192])
def test_row_strides_and_no_mass(ops, dev, ld):
    rng = np.random.default_rng(ld)
    logits = (rng.standard_normal((7, 5001)) * 3000).astype(np.int32)
    rules = random_rules(rng, 7, 5001, 1000.0)
    check(ops, dev, logits, rules, ld=ld)
    tokens, mass = run(ops, dev, logits, rules, ld=ld, mass=False)
    assert (mass == LEFT).all() and (tokens == run(ops, dev, logits, rules, ld=ld)[0]).all()


def test_draws_follow_the_weights(ops, dev):
    """Random numbers at equal steps over [0, 2^32) draw each token as often as its weight says, to within one."""
    v, n = 300, 2048
    x = (np.random.default_rng(2).standard_normal(v) * 2000).astype(np.int32)
    tokens, mass = run(ops, dev, np.tile(x, (n, 1)), [rule(1000.0, top_k=40, random=i * ((1 << 32) // n)) for i in range(n)])
    got = np.bincount(tokens, minlength=v)
    for t in np.unique(tokens):
        w, total = mass[np.nonzero(tokens == t)[0][0]]
        assert abs(got[t] - n * w / total) <= 1
    assert len(np.unique(tokens)) > 5


def test_many_rows(ops, dev):
    rng = np.random.default_rng(11)
    logits = (rng.standard_normal((700, 1500)) * 3000).astype(np.int32)
    check(ops, dev, logits, random_rules(rng, 700, 1500, 1000.0))


def test_behind_the_token_rules(ops, dev):
    """Penalties, biases and a mask by sslm_hip_pick_tokens, then sampling from its adjusted logits."""
    rng = np.random.default_rng(21)
    rows, v = 6, 7001
    logits = (rng.standard_normal((rows, v)) * 3000).astype(np.int32)
    hist = [rng.integers(0, v, 50).astype(np.int32) for _ in range(rows)]
    ids, vals = [rng.integers(0, v, 8).astype(np.int32) for _ in range(rows)], [rng.integers(-9000, 9000, 8).astype(np.int32) for _ in range(rows)]
    keep = [dev.upload(x) for x in (*hist, *ids, *vals)]
    table = (LogitRule * rows)()
    for r in range(rows):
        table[r] = LogitRule(keep[r].ptr, keep[rows + r].ptr, keep[2 * rows + r].ptr, None, 50, 8, 80000, 30, 20, 0)
    rules = random_rules(rng, rows, v, 1000.0)
    samp = (Sampling * rows)(*[Sampling(None, x["q_ln2"], x["q_b"], x["q_c"], x["top_k"], x["top_p"], x["min_p"], x["random"]) for x in rules])
    d, t, st = dev.upload(logits), dev.upload(np.frombuffer(bytes(table), np.uint8)), dev.upload(np.frombuffer(bytes(samp), np.uint8))
    best, tokens, mass = dev.zeros(rows, np.int32), dev.zeros(rows, np.int32), dev.zeros((rows, 2), np.int64)
    n, m = ops.pick_workspace(rows, v), ops.sample_workspace(rows, v)
    w0, w1 = dev.zeros(n, np.uint8), dev.zeros(m, np.uint8)
    ops.pick_tokens(rows=rows, vocab=v, logits=d.ptr, rules=t.ptr, tokens=best.ptr, adjusted=d.ptr, workspace=w0.ptr, workspace_bytes=n)()
    ops.sample_tokens(rows=rows, vocab=v, logits=d.ptr, rules=st.ptr, tokens=tokens.ptr, mass=mass.ptr, workspace=w1.ptr, workspace_bytes=m)()
    assert ops.lib.lib.sslm_hip_synchronize() == 0
    adjusted = d.numpy()
    assert (adjusted != logits).any()
    for r, x in enumerate(rules):
        want = ref.sample(adjusted[r], None, *[x[k] for k in ("q_ln2", "q_b", "q_c", "top_k", "top_p", "min_p", "random")])
        assert (tokens.numpy()[r], *mass.numpy()[r]) == want
        if x["top_k"] == 1:
            assert tokens.numpy()[r] == best.numpy()[r]


def test_sampling_record_layout():
    assert ctypes.sizeof(Sampling) == 48
