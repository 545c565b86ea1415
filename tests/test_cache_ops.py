"""What the paged cache's and the sampling's entries refuse before they launch anything (no GPU is touched), and the
definitions the GPU tests compare against, against plainer ones."""
import ctypes

import numpy as np
import pytest

import cache_ops_ref as ref
from superslm_amd.batch_ops import BatchOps, SampleArgs, Sampling, sampling_constants
from superslm_amd.cache_ops import CacheAttentionArgs, CacheCompactArgs, CacheOps, CacheStoreArgs, CacheUpdateArgs

INVALID, SMALL, MISALIGNED = 1, 2, 3
ANY = 1 << 20  # a non-null, aligned address that no refused call reads


@pytest.fixture(scope="module")
def cache(hip_lib):
    return CacheOps(hip_lib)


@pytest.fixture(scope="module")
def batch(hip_lib):
    return BatchOps(hip_lib)


def test_struct_sizes():
    assert [ctypes.sizeof(t) for t in (CacheUpdateArgs, CacheCompactArgs, CacheStoreArgs, CacheAttentionArgs, Sampling, SampleArgs)] == \
        [112, 88, 256, 224, 48, 56]


PAGES = dict(rows=3, pages=20, page_tokens=16, table_ld=8, pool=ANY, page_bytes=64, tables=ANY, lengths=ANY, new_tables=ANY, result=ANY,
             workspace=ANY, workspace_bytes=1 << 40)
REFUSED_PAGES = [
    ({"rows": 0}, INVALID), ({"rows": 4097}, INVALID), ({"pages": 0}, INVALID), ({"pages": (1 << 18) + 1}, INVALID), ({"table_ld": 0}, INVALID),
    ({"table_ld": (1 << 20) + 1}, INVALID), *[({"page_tokens": x}, INVALID) for x in (0, 1, 8, 24, 48, 512, -16)], ({"page_bytes": 0}, INVALID),
    ({"page_bytes": 72}, INVALID), ({"page_bytes": -64}, INVALID), ({"page_bytes": 1 << 50}, INVALID), ({"pool": ANY + 8}, INVALID),
    *[({k: None}, INVALID) for k in ("pool", "tables", "lengths", "new_tables", "result", "workspace")],
    ({"workspace": ANY + 16}, MISALIGNED), ({"workspace_bytes": 100}, SMALL)]


@pytest.mark.parametrize("change,status", REFUSED_PAGES + [({k: None}, INVALID) for k in ("source", "keep", "room", "new_lengths")])
def test_update_refusals(change, status, cache):
    assert cache.update(**dict(PAGES, source=ANY, keep=ANY, room=ANY, new_lengths=ANY, **{}) | change)(raw=True) == status


@pytest.mark.parametrize("change,status", REFUSED_PAGES + [({"map": None}, INVALID)])
def test_compact_refusals(change, status, cache):
    assert cache.compact(**dict(PAGES, map=ANY) | change)(raw=True) == status


LAYER = dict(rows=3, tokens=9, max_new=4, heads=4, kv_heads=2, head_dim=64, pages=20, page_tokens=16, table_ld=8, pool=ANY, page_bytes=4112,
             k_offset=0, v_offset=2048, exp_offset=4096, tables=ANY, row_tokens=ANY, row_start=ANY)
REFUSED_LAYER = [
    ({"rows": 0}, INVALID), ({"rows": 65536}, INVALID), ({"tokens": 0}, INVALID), ({"max_new": 0}, INVALID), ({"max_new": 10}, INVALID),
    ({"heads": 5}, INVALID), ({"heads": 0}, INVALID), ({"kv_heads": 0}, INVALID), ({"head_dim": 48}, INVALID), ({"heads": 130}, INVALID),
    ({"pages": 0}, INVALID), ({"page_tokens": 20}, INVALID), ({"page_tokens": 64}, INVALID), ({"table_ld": 0}, INVALID), ({"page_bytes": 4104}, INVALID),
    ({"page_bytes": 4096}, INVALID), ({"k_offset": -16}, INVALID), ({"k_offset": 8}, INVALID), ({"v_offset": 2080}, INVALID), ({"exp_offset": 4109}, INVALID),
    ({"exp_offset": -1}, INVALID), ({"pool": ANY + 4}, INVALID), *[({k: None}, INVALID) for k in ("pool", "tables", "row_tokens", "row_start")]]


@pytest.mark.parametrize("change,status", REFUSED_LAYER + [
    ({"rope_dim": 4}, INVALID), ({"rope_dim": -8}, INVALID), ({"rope_dim": 72}, INVALID), ({"rope_rows": 0}, INVALID), ({"rope_cos": None}, INVALID),
    ({"rope_sin": None}, INVALID), ({"q_ld": 255}, INVALID), ({"k_ld": 127}, INVALID), ({"v_ld": 0}, INVALID), ({"q_out": None}, INVALID),
    ({"q_out": ANY, "q": ANY, "q_ld": 300}, INVALID),
    *[({k: None}, INVALID) for k in ("k", "v", "k_scale", "v_scale", "r_t_k", "e_t_k", "r_t_v", "e_t_v", "clamped", "status")]])
def test_store_refusals(change, status, cache):
    f = dict(LAYER, rope_dim=64, rope_halves=0, rope_rows=100, rope_cos=ANY, rope_sin=ANY, q=ANY, k=ANY, v=ANY, k_scale=ANY, v_scale=ANY, r_t_k=ANY,
             e_t_k=ANY, r_t_v=ANY, e_t_v=ANY, q_out=ANY + 4096, clamped=ANY, status=ANY)
    assert cache.store(**f | change)(raw=True) == status


@pytest.mark.parametrize("change,status", REFUSED_LAYER + [
    ({"max_width": 0}, INVALID), ({"max_width": (1 << 24) + 1}, INVALID), ({"q": ANY + 8}, INVALID), ({"workspace": ANY + 64}, MISALIGNED),
    ({"workspace_bytes": 64}, SMALL),
    *[({k: None}, INVALID) for k in ("q", "q_scale", "khead_m", "khead_e", "ctx_fold", "codes", "scales", "status", "workspace")]])
def test_attention_refusals(change, status, cache):
    f = dict(LAYER, max_width=100, q=ANY, q_scale=ANY, khead_m=ANY, khead_e=ANY, ln2_q=1, b_q=1, ca_q=1, ctx_fold=ANY, site=(1 << 30, 0), codes=ANY,
             scales=ANY, status=ANY, workspace=ANY, workspace_bytes=1 << 40)
    assert cache.attention(**f | change)(raw=True) == status


@pytest.mark.parametrize("change,status", [
    ({"rows": 0}, INVALID), ({"rows": 65536}, INVALID), ({"vocab": 0}, INVALID), ({"vocab": (1 << 24) + 1}, INVALID), ({"logits_ld": 99}, INVALID),
    ({"logits_ld": 0}, INVALID), ({"logits": ANY + 2}, INVALID), *[({k: None}, INVALID) for k in ("logits", "rules", "tokens", "workspace")],
    ({"workspace": ANY + 8}, MISALIGNED), ({"workspace_bytes": 7}, SMALL)])
def test_sample_refusals(change, status, batch):
    f = dict(rows=2, vocab=100, logits=ANY, rules=ANY, tokens=ANY, mass=ANY, workspace=ANY, workspace_bytes=1 << 30)
    assert batch.sample_tokens(**f | change)(raw=True) == status


def test_a_struct_of_another_size_is_refused(cache, batch):
    calls = [cache.update(**PAGES, source=ANY, keep=ANY, room=ANY, new_lengths=ANY), cache.compact(**PAGES, map=ANY),
             batch.sample_tokens(rows=2, vocab=100, logits=ANY, rules=ANY, tokens=ANY, mass=ANY, workspace=ANY, workspace_bytes=1 << 30)]
    for call in calls:
        call.args.struct_size -= 8
        assert call(raw=True) == INVALID


def test_workspaces_of_sizes_outside_the_domain_are_zero(cache, batch):
    assert cache.update_workspace(0, 1, 1) == cache.compact_workspace(1, 0, 1) == batch.sample_workspace(1, 0) == 0
    assert cache.attention_workspace(1, 1, 2, 4, 2, 64, 16, 10) == cache.attention_workspace(1, 1, 1, 4, 2, 64, 17, 10) == 0
    assert cache.update_workspace(4096, 1 << 18, 100) > 0 and cache.compact_workspace(1, 1, 1) > 0 and batch.sample_workspace(1, 1) > 0
    assert cache.attention_workspace(1, 1, 1, 4, 2, 64, 16, 1) > 0


@pytest.mark.parametrize("rows,tokens,max_new,heads,kv_heads,dim,width,fits", [
    (65535, 65535, 1, 256, 256, 32, 100, False), (32767, 32767, 1, 256, 256, 32, 100, True),  # a block of 512 threads per (row, KV head)
    (65535, 65535, 1, 64, 64, 128, 100, True), (65535, 65535, 1, 256, 128, 32, 100, True),
    (1, (1 << 31) - 1, 2, 256, 1, 32, 100, False), (1, (1 << 31) - 1, 1, 256, 1, 32, 100, True),  # 64 query rows to a block of 256
    (1, 1 << 23, 2, 256, 1, 32, 100, False), (1, 1 << 21, 2, 256, 1, 32, 100, False), (1, 1 << 18, 2, 256, 1, 32, 100, True),
    (1, 1 << 23, 1 << 22, 1, 1, 32, 100, False), (1, 1 << 23, (1 << 22) - 1, 1, 1, 32, 100, True)])
def test_attention_that_no_launch_holds_has_no_workspace(cache, rows, tokens, max_new, heads, kv_heads, dim, width, fits):
    n = cache.attention_workspace(rows, tokens, max_new, heads, kv_heads, dim, 16, width)
    assert (n >= tokens * heads * dim * 4) if fits else n == 0


@pytest.mark.parametrize("tokens,heads,width,fits", [(1 << 30, 256, 1 << 24, False), ((1 << 31) - 1, 256, 1 << 24, False), ((1 << 31) - 1, 128, 1 << 24, False),
                                                     (1 << 28, 256, 1 << 24, False), ((1 << 28) - 1, 256, 1 << 24, True), (1 << 30, 256, 3 << 20, True)])
def test_attention_whose_scores_pass_64_bits_of_bytes_has_no_workspace(cache, tokens, heads, width, fits):
    n = cache.attention_workspace(1, tokens, 1, heads, 1, 32, 16, width)
    assert (n >= tokens * heads * width * 4) if fits else n == 0


def test_an_unknown_field_or_a_number_too_large_is_an_error(cache):
    with pytest.raises(TypeError):
        cache.compact(**PAGES, map=ANY, colour=1)
    with pytest.raises(OverflowError):
        cache.compact(**PAGES | {"rows": 1 << 40}, map=ANY)


# ---- the definitions ----
def test_rounding_and_landing_against_fractions():
    from fractions import Fraction as F
    rng = np.random.default_rng(1)
    for _ in range(300):
        x, e = int(rng.integers(-40000, 40000)), int(rng.integers(0, 9))
        y = F(x, 1 << e)
        assert int(ref.round_away(x, e)) == (1 if x > 0 else -1) * int(abs(y) + F(1, 2))
        c, m, r, k = int(rng.integers(-127, 128)), int(rng.integers(-(1 << 31), 1 << 31)), int(rng.integers(1 << 31, 1 << 32)), int(rng.integers(40, 70))
        y = F(c * m * r, 1 << k)
        assert ref.land(c, m, 62 - k, r, 0) == (1 if y > 0 else -1) * int(abs(y) + F(1, 2))


def test_exponents_hold_their_values():
    for top in (0, 1, 127, 128, 254, 255, 509, 510, 16319, 16320, 32512):
        e = ref.need(np.array([top, -top]))
        assert ref.round_away(top, e) <= 127 and (e == 0 or ref.round_away(top, e - 1) > 127) and e <= 8


def test_sampling_against_a_list_of_weights():
    """Token by token over an explicit list, without sorting tricks."""
    rng = np.random.default_rng(5)
    for trial in range(200):
        v = int(rng.integers(1, 40))
        x = rng.integers(-3000, 3000, v).astype(np.int32)
        c = sampling_constants(float(rng.uniform(50, 3000)))
        k, p, m, u = int(rng.integers(0, v + 2)), int(rng.integers(0, 65537)), int(rng.integers(0, 20000)), int(rng.integers(0, 1 << 32))
        items = sorted((-int(t), i) for i, t in enumerate(x))
        best = -items[0][0]
        w = []
        for t, i in items:
            d = best + t
            w.append((((c["q_b"] - d % c["q_ln2"]) ** 2 + c["q_c"]) >> (d // c["q_ln2"]) if d < 30 * c["q_ln2"] else 0, i))
        w = w[:k] if k else w
        total, run, cut = sum(a for a, _ in w), 0, []
        for a, i in w:
            if cut and run * 65536 >= total * p:
                break
            cut.append((a, i))
            run += a
        kept = [(a, i) for a, i in cut if a * 65536 >= m * (c["q_b"] ** 2 + c["q_c"])]
        total, run = sum(a for a, _ in kept), 0
        for a, i in kept:
            run += a
            if run > total * u >> 32:
                break
        assert ref.sample(x, None, c["q_ln2"], c["q_b"], c["q_c"], k, p, m, u) == (i, a, total)


def test_the_weights_follow_the_exponential():
    """The i-exp is within 0.3 % of exp where it holds eight bits or more."""
    c = sampling_constants(45000.0)
    w0 = c["q_b"] ** 2 + c["q_c"]
    d = np.arange(0, 8 * 45000, 977)
    w = [((c["q_b"] - int(x) % c["q_ln2"]) ** 2 + c["q_c"]) >> (int(x) // c["q_ln2"]) for x in d]
    assert (np.abs(np.array(w) / w0 / np.exp(-d / 45000.0) - 1) < 4e-3).all()
