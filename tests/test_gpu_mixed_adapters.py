"""Decode steps whose sequences have different adapters, or none, run as one launch sequence: tokens
and KV against the C oracle with each sequence's own adapter."""
import numpy as np
import pytest

from adapter_view import AdapterView
from conftest import synthetic
from oracle_bind import OracleModel
from superslm_amd.sslm import Model
from superslm_amd.sslm_artifact import PEFT_PROJECTIONS, build_adapter

pytestmark = pytest.mark.gpu


def adapters(sm):
    """Ranks and projections that differ: some of every kind, one of a single layer, odd and full ranks."""
    return [build_adapter(sm, rank=16, targets=("q_proj", "v_proj"), seed=1),
            build_adapter(sm, rank=5, targets=PEFT_PROJECTIONS, seed=2),
            build_adapter(sm, rank=64, targets=("o_proj", "down_proj", "gate_proj"), layers=[0], seed=3),
            build_adapter(sm, rank=1, targets=("k_proj", "up_proj"), seed=4)]


class Requests:
    """The same requests on the backend and on the oracle; `which[i]`: sequence i's adapter or None."""

    def __init__(self, hip_lib, oracle_lib, sm, art, which):
        self.blobs = adapters(sm)
        self.model = Model(hip_lib, art)
        self.ads = [self.model.adapter(b) for b in self.blobs]
        self.pool = self.model.pool(len(which))
        self.views = [AdapterView(b) for b in self.blobs]
        self.oracle = {a: OracleModel(oracle_lib, sm, adapter=None if a is None else self.views[a]) for a in [None, 0, 1, 2, 3]}
        self.seqs, self.want = [], []
        rng = np.random.default_rng(len(which))
        for i, a in enumerate(which):
            prompt = rng.integers(0, sm.config.vocab, size=2 + i % 7)
            s = self.pool.seq()
            s.set_adapter(None if a is None else self.ads[a])
            s.prefill(prompt)
            o = self.oracle[a].new_seq()
            assert o.prefill(prompt) == (0, len(prompt))
            self.seqs.append(s)
            self.want.append(o)

    def attach(self, i, a):
        self.seqs[i].set_adapter(None if a is None else self.ads[a])
        self.want[i].om = self.oracle[a]

    def step(self, budget, order=None):
        order = range(len(self.seqs)) if order is None else order
        got = self.model.decode_step([self.seqs[i] for i in order], budget)
        for i, t in zip(order, got):
            st, tok = self.want[i].decode_step(budget)
            assert st == 0 and t == tok, (i, t, tok)

    def close(self):
        # the pool hands out its last block first
        for i, o in enumerate(self.want):
            assert np.array_equal(self.pool.kv_block(len(self.want) - 1 - i), o.kv), f"KV of sequence {i}"
        for s in self.seqs:
            s.release()
        for a in self.ads:
            a.release()
        self.pool.close()
        self.model.close()


@pytest.mark.parametrize("name,which", [
    ("tiny", [0, 1]),
    ("small", [None, 2, 1, 0, 3, None, 1]),
    ("medium", [3, None, 0, 1, 2]),
    ("tiny", [(None, 0, 1, 2, 3)[i % 5] for i in range(37)]),
    ("tiny", [(None, 0, 1, 2, 3)[i * 7 % 5] for i in range(73)]),
    ("tiny", [(0, 1, 2, 3)[i % 4] for i in range(130)]),  # more than one launch sequence
])
@pytest.mark.parametrize("budget", [None, 1])
def test_mixed_adapters_match_the_oracle(name, which, budget, hip_lib, oracle_lib):
    sm, art = synthetic(name)
    print(f"case mixed adapters {name} x {len(which)} budget {budget}", flush=True)
    r = Requests(hip_lib, oracle_lib, sm, art, which)
    layers = sm.config.layers
    r.step(layers)  # the prompts' first tokens
    for _ in range(3 * (1 if budget is None else layers)):
        r.step(budget or layers)
    r.close()


def test_adapters_change_places_between_steps(hip_lib, oracle_lib):
    """The same graph replays with other adapters on the rows, then with one on all of them, then none."""
    sm, art = synthetic("tiny")
    r = Requests(hip_lib, oracle_lib, sm, art, [0, 1, None, 2, 3, 1])
    layers = sm.config.layers
    for which in ([0, 1, None, 2, 3, 1], [1, 0, 3, None, 2, 2], [1] * 6, [None] * 6, [2, 2, 0, 1, None, 3]):
        print(f"case swap {which}", flush=True)
        for i, a in enumerate(which):
            r.attach(i, a)
        r.step(layers)
        r.step(layers, order=[5, 3, 1, 0, 2, 4])
    r.close()


def test_sequences_at_different_layers(hip_lib, oracle_lib):
    """Half the sequences one layer ahead: two launch sequences, each with several adapters."""
    sm, art = synthetic("small")
    r = Requests(hip_lib, oracle_lib, sm, art, [0, 1, 2, None, 3, 1])
    r.step(sm.config.layers)
    r.step(1, order=[0, 2, 4])
    print("case layers", flush=True)
    for _ in range(5):
        r.step(1)
    r.close()
