"""Shared prompts (sslm_prefix_*, sslm_seq_adopt_prefix): tokens, KV and blobs of sequences that adopt
one against the oracle's sequences that take the prompt themselves, with the decode attention over shared
prompts forced on and off; and a batch that joins prefixes, adapters and token rules."""
import numpy as np
import pytest

from adapter_view import AdapterView, with_delta_exponent
from oracle_bind import OracleModel
from superslm_amd.sslm import Model
from superslm_amd.sslm_artifact import CONFIGS, ModelConfig, build_adapter, build_synthetic, with_weight_rows

pytestmark = pytest.mark.gpu

INVALID, FROZEN, SCHEMA_MISMATCH, POOL_LIVE = 1, 13, 21, 9
SHAPES = {
    "tiny": CONFIGS["tiny"], "medium": CONFIGS["medium"],
    # four KV heads of one query head: past 512 positions the split attention; three KV heads: always it
    "kv4": ModelConfig(hidden=256, layers=2, heads=4, kv_heads=4, head_dim=64, inter=512, vocab=512, context_cap=900, tie_embeddings=True),
    "kv3": ModelConfig(hidden=384, layers=2, heads=6, kv_heads=3, head_dim=64, inter=512, vocab=512, context_cap=300,
                       tie_embeddings=False, with_bias=True),
    # head size 256, 16 query heads to a KV head
    "wide": ModelConfig(hidden=4096, layers=1, heads=16, kv_heads=1, head_dim=256, inter=512, vocab=512, context_cap=200, tie_embeddings=True),
}
_MODELS = {}


def built(name):
    if name not in _MODELS:
        _MODELS[name] = build_synthetic(SHAPES[name], seed=11)
    return _MODELS[name]


class Batch:
    """Sequences over prefixes on the backend, each beside an oracle sequence with the whole prompt.
    members: (prefix index or None, own prompt's length, adapter index or None)."""

    def __init__(self, hip_lib, oracle_lib, sm, lengths, members, blobs=()):
        self.sm, c = sm, sm.config
        self.model = Model(hip_lib, sm.to_array())
        self.ads = [self.model.adapter(b) for b in blobs]
        om = {None: OracleModel(oracle_lib, sm)}
        views = [AdapterView(b) for b in blobs]
        om.update({i: OracleModel(oracle_lib, sm, adapter=v) for i, v in enumerate(views)})
        self.pool = self.model.pool(len(lengths) + len(members))
        rng = np.random.default_rng(sum(lengths) + len(members))
        self.prefixes, prompts = [], []
        for n in lengths:
            p = self.pool.prefix()
            prompt = rng.integers(0, c.vocab, size=n)
            cut = n // 3
            if cut:
                p.prefill(prompt[:cut])  # in two calls
            p.prefill(prompt[cut:])
            p.freeze()
            self.prefixes.append(p)
            prompts.append(prompt)
        self.seqs, self.want = [], []
        for pre, n, ad in members:
            s, o, own = self.pool.seq(), om[None].new_seq(), rng.integers(0, c.vocab, size=n)
            if pre is not None:
                s.adopt(self.prefixes[pre])
                assert o.prefill(prompts[pre]) == (0, len(prompts[pre]))
            if ad is not None:
                s.set_adapter(self.ads[ad])
                o.om = om[ad]
            if n:
                s.prefill(own)
                assert o.prefill(own) == (0, n)
            self.seqs.append(s)
            self.want.append(o)

    def step(self, budget=None, order=None):
        budget = budget or self.sm.config.layers
        order = list(range(len(self.seqs))) if order is None else order
        got = self.model.decode_step([self.seqs[i] for i in order], budget)
        for i, t in zip(order, got):
            assert self.want[i].decode_step(budget) == (0, t), i

    def check_kv(self):
        total = len(self.prefixes) + len(self.seqs)
        for i, o in enumerate(self.want):  # the pool hands out its last block first, the prefixes' ahead
            assert np.array_equal(self.pool.kv_block(total - 1 - len(self.prefixes) - i), o.kv), f"KV of sequence {i}"

    def close(self):
        for s in self.seqs:
            s.release()
        for p in self.prefixes:
            p.release()
        for a in self.ads:
            a.release()
        self.pool.close()
        self.model.close()


@pytest.mark.parametrize("name,lengths,members", [
    ("tiny", [20], [(0, 0, None), (0, 3, None), (0, 1, None)]),
    ("tiny", [17, 31], [(1, 2, None), (None, 5, None), (0, 4, None), (1, 0, None), (0, 1, None), (None, 1, None)]),
    ("medium", [40, 1], [(0, 1, None), (1, 9, None), (0, 7, None)]),
    ("kv4", [700], [(0, 3, None), (0, 0, None), (0, 40, None), (None, 30, None)]),
    ("kv4", [333, 64], [(0, 5, None), (1, 70, None), (0, 64, None)]),
    ("kv3", [130, 95], [(i % 2, 1 + i, None) for i in range(19)]),
    ("wide", [150], [(0, 4, None), (0, 1, None)]),
])
@pytest.mark.parametrize("shared", ["1", "0"])
@pytest.mark.parametrize("budget", [None, 1])
def test_adopted_prefix_matches_the_oracle(name, lengths, members, shared, budget, hip_lib, oracle_lib, monkeypatch):
    monkeypatch.setenv("SSLM_HIP_SHARED_ATTN", shared)
    print(f"case prefix {name} {lengths} x {len(members)} shared={shared} budget={budget}", flush=True)
    b = Batch(hip_lib, oracle_lib, built(name), lengths, members)
    b.step()  # the prompts' first tokens: logits only
    for _ in range(4 * (1 if budget is None else b.sm.config.layers)):
        b.step(budget)
    b.check_kv()
    b.close()


def test_prefix_graph_replays_over_a_growing_context(hip_lib, oracle_lib, monkeypatch):
    """One recorded step replayed while the own parts grow past a tile and past the recorded sizes, the
    members in another order, some left out."""
    monkeypatch.setenv("SSLM_HIP_SHARED_ATTN", "1")
    b = Batch(hip_lib, oracle_lib, built("kv4"), [90, 200], [(0, 2, None), (1, 3, None), (0, 250, None), (None, 4, None)])
    b.step()
    print("case growing", flush=True)
    for i in range(24):
        b.step(order=[[0, 1, 2, 3], [3, 2, 1, 0], [2, 0, 1]][i % 3])
    b.check_kv()
    b.close()


def test_prefix_with_adapters_and_rules(hip_lib, oracle_lib, monkeypatch):
    """What a server's batch holds at once: a shared prompt, adapters that differ, token rules on some.
    The same requests one by one, on sequences that took the prompt themselves, give the same tokens."""
    monkeypatch.setenv("SSLM_HIP_SHARED_ATTN", "1")
    sm = built("kv3")
    blobs = [build_adapter(sm, rank=16, targets=("q_proj", "v_proj"), seed=1),
             build_adapter(sm, rank=7, targets=("o_proj", "down_proj", "k_proj"), seed=2)]
    rules = [None, {"repetition": 1.4}, {"bias": [(i, 50000) for i in range(0, 512, 7)]}, {"presence": 30000, "frequency": 8000}]
    model = Model(hip_lib, sm.to_array())
    ads = [model.adapter(x) for x in blobs]
    pool = model.pool(14)
    rng = np.random.default_rng(4)
    prompt, owns = rng.integers(0, 512, size=120), [rng.integers(0, 512, size=1 + i % 5) for i in range(12)]

    def request(i, s):
        a = (None, 0, 1)[i % 3]
        if a is not None:
            s.set_adapter(ads[a])
        if rules[i % 4]:
            s.set_rules(**rules[i % 4])
        s.prefill(owns[i])

    prefix = pool.prefix()
    prefix.prefill(prompt)
    prefix.freeze()
    seqs = []
    for i in range(12):
        s = pool.seq()
        s.adopt(prefix)
        request(i, s)
        seqs.append(s)
    prefix.release()  # lives on with its adopters
    print("case joined", flush=True)
    together = [model.decode_step(seqs, 2) for _ in range(6)]
    for i, s in enumerate(seqs):
        blob = s.save()
        s.release()
        alone = pool.seq()
        alone.prefill(prompt)
        request(i, alone)
        assert [model.decode_step([alone], 2)[0] for _ in range(6)] == [t[i] for t in together], i
        assert alone.save() == blob, i
        alone.release()
    for a in ads:
        a.release()
    pool.close()
    model.close()


BAD = 5


@pytest.mark.parametrize("kind", ["zero", "attention"])
@pytest.mark.parametrize("budget", [2, 1])
def test_a_refusal_inside_a_shared_batch(kind, budget, hip_lib, monkeypatch):
    """The second of three adopters refuses: before the attention (its pending token's embedding is zero;
    a bias made it the pick), or in the attention (an adapter swells its q scale until the i-exp has no
    constant).  Statuses, tokens and blobs as without sharing: the first advances, the third is untouched."""
    def edit(m):
        for h in range(3):
            sm_, e = m.consts[f"layer0.softmax_khead{h}"]
            m.consts[f"layer0.softmax_khead{h}"] = (sm_, e + 10)

    sm = build_synthetic(SHAPES["kv3"], seed=11, edit=edit)
    art = with_weight_rows(sm, "embed", {BAD: np.zeros(sm.config.hidden, np.int8)}) if kind == "zero" else sm.to_bytes()
    blob = with_delta_exponent(build_adapter(sm, rank=16, targets=("q_proj",), seed=3), -14) if kind == "attention" else None
    seen = {}
    for shared in ("0", "1"):
        monkeypatch.setenv("SSLM_HIP_SHARED_ATTN", shared)
        model = Model(hip_lib, art)
        pool = model.pool(4)
        ad = model.adapter(blob) if blob else None
        p = pool.prefix()
        p.prefill([(i * 37 + 11) % 512 for i in range(140)])
        p.freeze()
        seqs = [pool.seq() for _ in range(3)]
        for s in seqs:
            s.adopt(p)
        if kind == "zero":
            seqs[1].set_rules(bias=[(BAD, 1 << 30)])
        else:
            seqs[1].set_adapter(ad)
        print(f"case refusal {kind} budget={budget} shared={shared}", flush=True)
        log = [model.decode_step(seqs, budget, raw=True)]  # the first tokens
        for _ in range(3):
            log.append(model.decode_step(seqs, budget, raw=True))
            log.append([s.save() for s in seqs])
        seen[shared] = log
        for s in seqs:
            s.release()
        p.release()
        if ad:
            ad.release()
        pool.close()
        model.close()
    assert seen["0"][1][0] != 0, "nothing refused"
    assert seen["0"] == seen["1"]


def test_prefix_refusals(hip_lib):
    schemas = [("a", {0: {t: 0 for t in range(0, 512, 2)}}, [0])]
    sm = build_synthetic(CONFIGS["tiny"], seed=7, schemas=schemas)
    model = Model(hip_lib, sm.to_bytes())
    pool, other = model.pool(4), model.pool(1)
    L = model.lib.lib
    p, s = pool.prefix(), pool.seq()
    assert p.prefill([1, 2, 3], raw=True) == (0, 3)
    assert s.adopt(p, raw=True) == INVALID  # not frozen
    p.freeze()
    p.freeze()
    assert p.prefill([4], raw=True) == (FROZEN, 0)
    assert p.set_schema(None) == FROZEN
    far = other.seq()
    assert far.adopt(p, raw=True) == INVALID  # another pool
    used = pool.seq()
    used.prefill([9])
    assert used.adopt(p, raw=True) == INVALID  # holds context
    st, schema = model.schema("a")
    bound = pool.seq()
    assert bound.set_schema(schema) == 0 and bound.adopt(p, raw=True) == SCHEMA_MISMATCH
    assert s.adopt(p, raw=True) == 0 and s.adopt(p, raw=True) == INVALID
    assert L.sslm_prefix_prefill(model.handle, None, None, 0, 1, 0, None, None) == INVALID
    assert L.sslm_prefix_release(None) == INVALID and L.sslm_seq_adopt_prefix(s.handle, None) == INVALID
    h = p.handle
    p.release()  # s still reads it
    assert L.sslm_prefix_release(h) == INVALID
    bound.release()
    fresh = pool.seq()
    assert L.sslm_seq_adopt_prefix(fresh.handle, h) == INVALID
    assert model.decode_step([s], 2)[0] >= 0
    for x in (fresh, used, far, s):
        x.release()  # s, the last adopter, takes the prefix down
    again = [pool.seq() for _ in range(4)]  # every block is free again
    for x in again:
        x.release()
    other.close()
    pool.close()
    model.close()


def test_a_released_prefix_is_refused_everywhere(hip_lib):
    model = Model(hip_lib, build_synthetic(CONFIGS["tiny"], seed=7).to_bytes())
    pool = model.pool(2)
    L = model.lib.lib
    p, s = pool.prefix(), pool.seq()
    h = p.handle
    p.prefill([1, 2, 3])
    p.freeze()
    p.release()  # nobody adopted it: it is gone
    assert L.sslm_prefix_release(h) == INVALID and L.sslm_prefix_freeze(h) == INVALID
    assert L.sslm_prefix_set_schema(h, None) == INVALID and L.sslm_seq_adopt_prefix(s.handle, h) == INVALID
    assert L.sslm_prefix_prefill(model.handle, h, None, 0, 1, 0, None, None) == INVALID
    s.prefill([1])
    assert model.decode_step([s], 2)[0] >= 0
    s.release()
    pool.close()
    model.close()


def test_shared_attention_over_prompts_of_growing_length(hip_lib, oracle_lib, monkeypatch):
    """Units whose scratch grows from step to step while graphs of the smaller ones are kept and run again."""
    monkeypatch.setenv("SSLM_HIP_SHARED_ATTN", "1")
    batch = Batch(hip_lib, oracle_lib, built("kv4"), [5, 64, 65, 300, 520], [(i, 2, None) for i in range(5)] + [(4, 1, None)])
    for _ in range(2):
        for order in ([0], [0, 1], [2, 1], [3, 0], [4, 5], [0, 1, 2, 3, 4, 5], [0], [3, 0], [0, 1]):
            batch.step(order=order)
    batch.check_kv()
    batch.close()


def test_prefix_under_a_schema_and_reset(hip_lib, oracle_lib):
    """The walk goes with the prefix; a reset sequence lets go of it and is a fresh one."""
    table = {0: {t: 1 for t in range(0, 512, 2)}, 1: {t: 0 for t in range(1, 512, 2)}}
    sm = build_synthetic(CONFIGS["tiny"], seed=7, schemas=[("ab", table, [0])])
    model = Model(hip_lib, sm.to_bytes())
    pool = model.pool(3)
    st, schema = model.schema("ab")
    p = pool.prefix()
    assert p.set_schema(schema) == 0
    p.prefill([10, 11, 12], kind=1)  # a schema-content span: the walk ends in state 1
    p.freeze()
    a, b = pool.seq(), pool.seq()
    for s in (a, b):
        assert s.set_schema(schema) == 0
    a.adopt(p)
    b.prefill([10, 11, 12], kind=1)
    toks = [model.decode_step([s], 2)[0] for s in (a, b)]
    assert toks[0] == toks[1] and toks[0] % 2 == 1
    assert a.save() == b.save()
    assert model.lib.lib.sslm_seq_reset(a.handle) == 0
    p.release()
    om = OracleModel(oracle_lib, sm).new_seq()
    a.set_schema(None)
    a.prefill([7, 8])
    om.prefill([7, 8])
    assert model.decode_step([a], 2)[0] == om.decode_step(2)[1]
    a.release()
    b.release()
    pool.close()
    model.close()
