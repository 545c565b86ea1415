"""Decoding under token rules (sslm_hip_seq_set_rules): every pick against the oracle's logits with the
rules applied in Python's integers."""
import ctypes

import numpy as np
import pytest

from batch_ops_ref import pick_row
from conftest import synthetic
from oracle_bind import OracleModel, Scale, _p, i8p, i32p
from superslm_amd.sslm import Model
from superslm_amd.sslm_artifact import CONFIGS, build_synthetic

pytestmark = pytest.mark.gpu
INVALID, ID_RANGE = 1, 15


class Ruled:
    """One sequence on the oracle, picked under rules and a schema's mask (its legal tokens, or None)."""

    def __init__(self, om, rules=None):
        self.o, self.rules, self.context, self.legal = om.new_seq(), rules, [], None

    def prefill(self, tokens):
        assert self.o.prefill(tokens) == (0, len(tokens))
        self.context += [int(t) for t in tokens]

    def step(self, budget):
        om, c, o = self.o.om, self.o.om.sm.config, self.o
        if o.ready_for_logits:
            o.ready_for_logits = False
        else:
            if o.state.layer_index == 0:
                sc = Scale()
                assert om.lib.or_embed_entry(ctypes.byref(om.m), o.current_token, _p(o.hidden, i8p), ctypes.byref(sc)) == 0
                o.state.scale = sc
            assert om.lib.or_run_layer_loop(ctypes.byref(om.m), ctypes.byref(o.state), budget, _p(o.kv, i8p)) == 0
            if o.state.layer_index < c.layers:
                return -1
        logits = np.zeros(c.vocab, np.int32)
        assert om.lib.or_final_logits(ctypes.byref(om.m), _p(o.hidden, i8p), _p(logits, i32p)) == 0
        r = self.rules or {}
        mask = None
        if self.legal is not None:
            mask = np.zeros((c.vocab + 7) // 8, np.uint8)
            for t in self.legal:
                mask[t >> 3] |= 1 << (t & 7)
        history = np.array(self.context if self.rules else [], np.int64)
        tok, _ = pick_row(logits, history, r.get("bias", []), mask, int(round(r.get("repetition", 1.0) * 65536)),
                          r.get("presence", 0), r.get("frequency", 0))
        o.current_token = tok
        o.state.layer_index = 0
        self.context.append(tok)
        return tok


RULES = [
    {"repetition": 1.3},
    {"presence": 30000, "frequency": 9000},
    None,
    {"repetition": 0.7, "frequency": -4000},
    {"bias": [(7, -10 ** 9), (11, 40000), (11, 40000), (300, -5)]},
    {"repetition": 2.0, "presence": 100000, "bias": [(i, 60000) for i in range(0, 512, 3)]},
]


@pytest.mark.parametrize("name", ["tiny", "small", "medium"])
@pytest.mark.parametrize("budget", [None, 1])
def test_rules_match_the_oracle(name, budget, hip_lib, oracle_lib):
    sm, art = synthetic(name)
    model, om = Model(hip_lib, art), OracleModel(oracle_lib, sm)
    pool = model.pool(len(RULES))
    rng = np.random.default_rng(3)
    seqs, want = [], []
    for i, r in enumerate(RULES):
        prompt = rng.integers(0, sm.config.vocab, size=3 + 2 * i)
        s, o = pool.seq(), Ruled(om, r)
        if r:
            s.set_rules(**r)
        s.prefill(prompt)
        o.prefill(prompt)
        seqs.append(s)
        want.append(o)
    L = sm.config.layers
    print(f"case rules {name} budget {budget}", flush=True)
    for _ in range(8 if budget is None else 4 * L):
        got = model.decode_step(seqs, budget or L)
        assert got == [o.step(budget or L) for o in want]
    for s in seqs:
        s.release()
    pool.close()
    model.close()


def test_rules_change_between_steps(hip_lib, oracle_lib):
    """Set on a running sequence (its whole context counts), changed, cleared; the sequence reset (its
    context counts no longer, its rules stay); prompts that pass over a produced token, until
    the counted tokens outnumber the context cap."""
    sm, art = synthetic("tiny")
    model, om = Model(hip_lib, art), OracleModel(oracle_lib, sm)
    pool = model.pool(2)
    L, rng = sm.config.layers, np.random.default_rng(5)
    seqs, want = [pool.seq(), pool.seq()], [Ruled(om), Ruled(om)]

    def step():
        assert model.decode_step(seqs, L) == [o.step(L) for o in want]

    def feed(n):
        for s, o in zip(seqs, want):
            p = rng.integers(0, sm.config.vocab, size=n)
            s.prefill(p)
            o.prefill(p)

    feed(5)
    step()
    step()
    for rules in ({"repetition": 1.5, "frequency": 20000}, {"bias": [(3, 10 ** 6)]}, None, {"presence": 50000}):
        print(f"case change {rules}", flush=True)
        if rules:
            seqs[1].set_rules(**rules)
        else:
            seqs[1].clear_rules()
        want[1].rules = rules
        step()
        step()
    seqs[1].prefill([])
    for s in seqs:
        s._pool_reset = s.pool.model.lib.lib.sslm_seq_reset(s.handle)
        assert s._pool_reset == 0
    want = [Ruled(om), Ruled(om, {"presence": 50000})]
    print("case reset", flush=True)
    feed(4)
    step()
    step()
    for _ in range(48):  # one token in, one produced and passed over
        feed(1)
        step()
    assert len(want[1].context) > sm.config.context_cap + 1
    for s in seqs:
        s.release()
    pool.close()
    model.close()


def test_rules_with_a_schema(hip_lib, oracle_lib):
    """Masked by the schema's page of the walk's state; a state without a legal token ends at -2."""
    table = {0: {t: (1 if t % 2 else 0) for t in range(0, 512, 5)}, 1: {t: 2 for t in range(40, 90)}, 2: {}}
    sm = build_synthetic(CONFIGS["tiny"], seed=7, schemas=[("s", table, [2])])
    model, om = Model(hip_lib, sm.to_bytes()), OracleModel(oracle_lib, sm)
    pool = model.pool(3)
    st, schema = model.schema("s")
    assert st == 0
    rules = [{"repetition": 1.4, "presence": 20000}, None, {"bias": [(t, 30000) for t in range(5, 512, 10)]}]
    seqs, want, walk = [], [], [0, 0, 0]
    for i, r in enumerate(rules):
        s, o = pool.seq(), Ruled(om, r)
        assert s.set_schema(schema) == 0
        if r:
            s.set_rules(**r)
        p = [9 + i, 100, 3 * i]
        s.prefill(p)
        o.prefill(p)
        seqs.append(s)
        want.append(o)
    L, live = sm.config.layers, [0, 1, 2]
    print("case schema", flush=True)
    for _ in range(6):
        got = model.decode_step([seqs[i] for i in live], L)
        for i, t in zip(list(live), got):
            legal = table[walk[i]]
            if not legal:
                assert t == -2
                live.remove(i)  # the reference refuses the next call of a dead end
                continue
            want[i].legal = sorted(legal)
            assert t == want[i].step(L), i
            walk[i] = legal[t]
        if not live:
            break
    for s in seqs:
        s.release()
    pool.close()
    model.close()


def test_rules_refusals(hip_lib):
    sm = build_synthetic(CONFIGS["tiny"], seed=7, damped_logit_scale=1.0 / 20000)
    model = Model(hip_lib, sm.to_bytes())
    pool = model.pool(1)
    s = pool.seq()
    assert s.set_rules(repetition=0.0, raw=True) == INVALID
    assert s.set_rules(repetition=-1.0, raw=True) == INVALID
    assert s.set_rules(bias=[(512, 1)], raw=True) == ID_RANGE
    assert s.set_rules(bias=[(-1, 1)], raw=True) == ID_RANGE
    assert model.lib.lib.sslm_hip_seq_set_rules(None, None) == INVALID
    s.prefill([1, 2, 3])
    s.set_rules(presence=5)
    p = model.decode_params(sm.config.layers, 1)
    st, out = model.decode_step([s], sm.config.layers, raw=True, params=p)
    assert st == INVALID
    s.clear_rules()
    assert model.decode_step([s], sm.config.layers, params=p)[0] >= 0
    s.release()
    pool.close()
    model.close()
