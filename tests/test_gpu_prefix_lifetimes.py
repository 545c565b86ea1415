"""Shared prompts across the lives of pools, prefixes and the threads that use them."""
import numpy as np
import pytest

from superslm_amd.sslm import Model
from superslm_amd.sslm_artifact import CONFIGS, build_synthetic

pytestmark = pytest.mark.gpu


def test_pools_of_other_sizes_follow_each_other(hip_lib, monkeypatch):
    """One model's pools, each destroyed before the next is made, so that a later and larger one may lie at an
    earlier one's address; the same batch of adopters in each has the same tokens and the same recorded shapes."""
    monkeypatch.setenv("SSLM_HIP_SHARED_ATTN", "1")
    sm = build_synthetic(CONFIGS["tiny"], seed=7)
    model = Model(hip_lib, sm.to_bytes())
    prompt = np.random.default_rng(3).integers(0, sm.config.vocab, size=20)
    seen = []
    for blocks in (3, 4, 9, 30, 3, 60, 5):
        print(f"case pool of {blocks}", flush=True)
        pool = model.pool(blocks)
        p = pool.prefix()
        p.prefill(prompt)
        p.freeze()
        seqs = [pool.seq() for _ in range(2)]
        for i, s in enumerate(seqs):
            s.adopt(p)
            s.prefill([5 + i])
        seen.append([model.decode_step(seqs, sm.config.layers) for _ in range(4)] + [s.save() for s in seqs])
        for s in seqs:
            s.release()
        p.release()
        pool.close()
    assert all(x == seen[0] for x in seen)
    model.close()
