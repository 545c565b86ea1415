"""What sampling's plan leaves at the start of the workspace, a record per row: it must not depend on the order in which a block's
waves run, as the token never does."""
import numpy as np
import pytest

import cache_ops_ref as ref
from superslm_amd.batch_ops import BatchOps, Sampling
from superslm_amd.device import Device
from test_gpu_sample import rule

pytestmark = pytest.mark.gpu

# SamplePlan of sample.hip
PLAN = np.dtype([("top", np.int32), ("sh", np.int32), ("state", np.int32), ("cut_k", np.int32), ("goal_k", np.uint32), ("a", np.uint32, 3),
                 ("b", np.uint32, 3), ("count", np.uint32), ("w", np.uint64, 2), ("kept", np.uint64, 2)])


@pytest.fixture(scope="module")
def ops(hip_lib):
    return BatchOps(hip_lib)


@pytest.fixture(scope="module")
def dev(hip_lib):
    return Device(hip_lib)


def plans(ops, dev, logits, rules, times=1):
    """The records after each of `times` calls; tokens and masses against the definition."""
    rows, v = logits.shape
    table = (Sampling * rows)(*[Sampling(None, x["q_ln2"], x["q_b"], x["q_c"], x["top_k"], x["top_p"], x["min_p"], x["random"]) for x in rules])
    d, t = dev.upload(logits), dev.upload(np.frombuffer(bytes(table), np.uint8))
    tokens, mass = dev.zeros(rows, np.int32), dev.zeros((rows, 2), np.int64)
    n = ops.sample_workspace(rows, v)
    ws, fill = dev.zeros(n, np.uint8), dev.upload(np.full(n, 0xA5, np.uint8))
    call = ops.sample_tokens(rows=rows, vocab=v, logits=d.ptr, logits_ld=v, rules=t.ptr, tokens=tokens.ptr, mass=mass.ptr, workspace=ws.ptr,
                             workspace_bytes=n)
    out = []
    for _ in range(times):
        dev.copy_device(ws, fill)
        call()
        assert ops.lib.lib.sslm_hip_synchronize() == 0
        out.append(np.frombuffer(ws.numpy()[:rows * PLAN.itemsize].tobytes(), PLAN))
    for r, x in enumerate(rules):
        want = ref.sample(logits[r], None, *[x[k] for k in ("q_ln2", "q_b", "q_c", "top_k", "top_p", "min_p", "random")])
        assert (tokens.numpy()[r], *mass.numpy()[r]) == want, r
    return out


@pytest.mark.parametrize("vocab", [20000, 151936])
def test_plans_of_equal_calls_are_equal(ops, dev, vocab):
    """Rules whose top-p leaves much less weight than the whole row's, with and without min-p: the draw's range follows from
    the narrowed weight, its tolerance from the whole one."""
    rng = np.random.default_rng(vocab)
    rows = 48
    logits = (rng.standard_normal((rows, vocab)) * 120000).astype(np.int32)
    rules = [rule(45000.0 * float(rng.uniform(0.6, 1.4)), (0, 300)[r % 2], int(rng.integers(6000, 60000)), (0, 40, 3000)[r % 3], int(rng.integers(0, 1 << 32)))
             for r in range(rows)]
    first, *others = plans(ops, dev, logits, rules, times=25)
    for p in others:
        for name in PLAN.names:
            assert (p[name] == first[name]).all(), name


def normal(rng, rows, vocab):
    return (rng.standard_normal((rows, vocab)) * 120000).astype(np.int32)


@pytest.mark.parametrize("vocab", [8193, 20000, 151936])
def test_ordinary_rows_are_drawn_without_the_search_over_the_row(ops, dev, vocab):
    """Spreads of 2.2 to 4.4 natural units: a result that only the search made right would show here."""
    rng = np.random.default_rng(vocab)
    rules = [rule(45000.0 * float(rng.uniform(0.6, 1.2)), *((40, 60000, 0), (0, 55000, 0), (300, 60000, 2000), (0, 65536, 0), (0, 65536, 500), (50, 65536, 0))[r % 6],
                  int(rng.integers(0, 1 << 32))) for r in range(36)]
    assert (plans(ops, dev, normal(rng, 36, vocab), rules)[0]["state"] == 0).all()


def test_rows_that_are_searched_whole(ops, dev):
    """Too many elements around a border for the list; and, found while gathering, too many of them in one slice."""
    rng = np.random.default_rng(7)
    flat = [rule(45000.0 * 6, 0, 58982, 0, int(rng.integers(0, 1 << 32))) for _ in range(6)]
    assert (plans(ops, dev, normal(rng, 6, 151936), flat)[0]["state"] == 1).all()
    x = np.full((3, 30000), -100000000, np.int32)
    x[:, 9000:11500] = 0
    side = [rule(1000.0, random=int(u)) for u in (0, 1 << 31, (1 << 32) - 1)]
    assert (plans(ops, dev, x, side)[0]["state"] == 2).all()
