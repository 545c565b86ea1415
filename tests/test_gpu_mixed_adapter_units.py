"""Decode calls of more sequences than one launch sequence holds, with and without adapters in any order: tokens,
KV and the order of refusals."""
import numpy as np
import pytest

from adapter_view import with_delta_exponent
from conftest import synthetic
from superslm_amd.sslm import Model
from superslm_amd.sslm_artifact import build_adapter, build_synthetic
from test_gpu_mixed_adapters import Requests
from test_gpu_prefix import SHAPES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", [
    [(None, 0)[i % 2] for i in range(256)],
    [(None, None, 1, None, 3)[i % 5] for i in range(150)],
    [None] * 140 + [2] + [None] * 3 + [0],
])
@pytest.mark.parametrize("budget", [None, 1])
def test_units_of_bare_and_adapted_sequences(which, budget, hip_lib, oracle_lib):
    sm, art = synthetic("tiny")
    print(f"case units x {len(which)} budget {budget}", flush=True)
    r = Requests(hip_lib, oracle_lib, sm, art, which)
    layers = sm.config.layers
    r.step(layers)  # the prompts' first tokens
    for _ in range(2 * (1 if budget is None else layers)):
        r.step(budget or layers)
    r.step(layers, order=list(range(len(which)))[::-1])
    r.close()


def test_a_refusal_among_several_units(hip_lib):
    """The call's 100th of 140 sequences refuses in its attention (its adapter swells the q scale until the i-exp has
    no constant), in a unit behind that of later, bare ones: the sequences ahead of it in the call advance as
    alone, those behind it stay as they were."""
    def edit(m):
        for h in range(3):
            sm_, e = m.consts[f"layer0.softmax_khead{h}"]
            m.consts[f"layer0.softmax_khead{h}"] = (sm_, e + 10)

    sm = build_synthetic(SHAPES["kv3"], seed=11, edit=edit)
    model = Model(hip_lib, sm.to_bytes())
    bad = model.adapter(with_delta_exponent(build_adapter(sm, rank=16, targets=("q_proj",), seed=3), -14))
    good = model.adapter(build_adapter(sm, rank=16, targets=("q_proj",), seed=4))
    pool, n, at = model.pool(141), 140, 100
    rng = np.random.default_rng(8)
    prompts = [rng.integers(0, 512, size=2 + i % 5) for i in range(n)]
    seqs = [pool.seq() for _ in range(n)]
    for i, s in enumerate(seqs):
        if i % 3 == 1 and i != at:
            s.set_adapter(good)
        s.prefill(prompts[i])
    first = model.decode_step(seqs, 2)
    seqs[at].set_adapter(bad)
    before = [s.save() for s in seqs]
    print("case refusal among units", flush=True)
    st, got = model.decode_step(seqs, 2, raw=True)
    assert st != 0
    after = [s.save() for s in seqs]
    assert after[at + 1:] == before[at + 1:]
    for i in (0, 1, 50, at - 1):
        alone = pool.seq()
        if i % 3 == 1:
            alone.set_adapter(good)
        alone.prefill(prompts[i])
        assert [model.decode_step([alone], 2)[0] for _ in range(2)] == [first[i], got[i]], i
        assert alone.save() == after[i], i
        alone.release()
    assert model.decode_step([seqs[i] for i in range(at + 1, n)], 2)  # and they go on
    for s in seqs:
        s.release()
    for a in (good, bad):
        a.release()
    pool.close()
    model.close()
