"""Shared prompts across the lives of pools, prefixes and the threads that use them."""
import struct
import threading
import time

import numpy as np
import pytest

from superslm_amd.sslm import Model
from superslm_amd.sslm_artifact import CONFIGS, ModelConfig, build_adapter, build_synthetic

pytestmark = pytest.mark.gpu

OK, INVALID, FROZEN = 0, 1, 13


def context_length(seq):
    return struct.unpack_from("<q", seq.save(), 60)[0]


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


def test_no_prefill_passes_a_freeze(hip_lib):
    """A long prefill holds the model; behind it wait a freeze, whose thread then adopts, and a prefill of the
    same prefix.  Whatever the order in which they get the model, the prefill is refused or ahead of the freeze:
    sequences that adopt right after the freeze and later have the same context."""
    cfg = ModelConfig(hidden=1024, layers=4, heads=8, kv_heads=2, head_dim=128, inter=2816, vocab=512, context_cap=6000,
                      tie_embeddings=True)
    model = Model(hip_lib, build_synthetic(cfg, seed=5).to_array())
    pool = model.pool(4)
    busy = pool.seq()
    long = np.random.default_rng(1).integers(0, cfg.vocab, size=6000)
    for turn in range(8):
        print(f"case freeze {turn}", flush=True)
        assert model.lib.lib.sslm_seq_reset(busy.handle) == 0
        p, early, late = pool.prefix(), pool.seq(), pool.seq()
        p.prefill([1, 2, 3])
        seen = {}

        def freeze():
            p.freeze()
            seen["adopt"] = early.adopt(p, raw=True)

        def extend():
            seen["extend"] = p.prefill([4, 5, 6, 7], raw=True)

        threads = [threading.Thread(target=f) for f in (lambda: busy.prefill(long, chunk_budget=len(long)), freeze, extend)]
        for t in threads:
            t.start()
            time.sleep(0.001)
        for t in threads:
            t.join(30)
            assert not t.is_alive()
        assert seen["adopt"] == OK and seen["extend"] in ((OK, 4), (FROZEN, 0))
        late.adopt(p)
        want = 7 if seen["extend"][0] == OK else 3
        assert (context_length(early), context_length(late)) == (want, want)
        a, b = (model.decode_step([s], cfg.layers) for s in (early, late))
        assert a == b
        for s in (early, late):
            s.release()
        p.release()
    busy.release()
    pool.close()
    model.close()


def test_prefix_verbs_against_a_release(hip_lib):
    """Every prefix verb while another thread releases the prefix: each takes effect or is refused, and when the
    adopters are gone every block is free again."""
    model = Model(hip_lib, build_synthetic(CONFIGS["tiny"], seed=7).to_bytes())
    L, pool = model.lib.lib, model.pool(5)
    statuses = set()
    for turn in range(60):
        print(f"case release {turn}", flush=True)
        p, seqs = pool.prefix(), [pool.seq() for _ in range(3)]
        h = p.handle
        p.prefill([1, 2, 3 + turn % 5])
        p.freeze()
        go = threading.Barrier(3)
        got = []

        def adopt():
            go.wait()
            for s in seqs:
                got.append(L.sslm_seq_adopt_prefix(s.handle, h))

        def others():
            go.wait()
            for _ in range(3):
                assert L.sslm_prefix_freeze(h) in (OK, INVALID)
                assert L.sslm_prefix_set_schema(h, None) in (FROZEN, INVALID)
                assert p.prefill([9], raw=True) in ((FROZEN, 0), (INVALID, 0))

        threads = [threading.Thread(target=f) for f in (adopt, others)]
        for t in threads:
            t.start()
        go.wait()
        assert L.sslm_prefix_release(h) == OK
        for t in threads:
            t.join(30)
            assert not t.is_alive()
        statuses.update(got)
        assert len(got) == 3 and set(got) <= {OK, INVALID} and got == sorted(got)  # none succeeds after a refusal
        adopters = [s for s, st in zip(seqs, got) if st == OK]
        if adopters:
            assert len({t for t in model.decode_step(adopters, 2)}) == 1
        for s in seqs:
            s.release()
        for s in [pool.seq() for _ in range(5)]:
            s.release()
    pool.close()
    model.close()


def test_a_sequence_with_an_adapter_does_not_adopt(hip_lib):
    """Its prompt's K/V would be without the adapter.  Refused, the sequence is still fresh: it takes the prompt
    itself, or adopts once the adapter is gone and may have it back for what follows."""
    sm = build_synthetic(CONFIGS["tiny"], seed=7)
    model = Model(hip_lib, sm.to_bytes())
    pool, prompt = model.pool(5), [7, 8, 9, 10]
    ad = model.adapter(build_adapter(sm, rank=16, targets=("q_proj", "k_proj", "v_proj"), seed=1))
    p = pool.prefix()
    p.prefill(prompt)
    p.freeze()
    a, b, plain = (pool.seq() for _ in range(3))  # blocks 3, 2 and 1
    print("case adapter before adoption", flush=True)
    for s in (a, b):
        s.set_adapter(ad)
        assert s.adopt(p, raw=True) == INVALID and context_length(s) == 0
    a.prefill(prompt)  # with its adapter
    plain.prefill(prompt)
    assert not np.array_equal(pool.kv_block(3), pool.kv_block(1))
    b.set_adapter(None)
    b.adopt(p)
    assert b.save() == plain.save()
    for s in (b, plain):
        s.set_adapter(ad)
        s.prefill([3, 4])
    assert [model.decode_step([b], 2) for _ in range(3)] == [model.decode_step([plain], 2) for _ in range(3)]
    assert b.save() == plain.save()
    for s in (a, b, plain):
        s.release()
    p.release()
    ad.release()
    pool.close()
    model.close()
