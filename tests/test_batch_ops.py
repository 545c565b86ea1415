"""What the batch operators' entries refuse before they launch anything (no GPU is touched)."""
import ctypes

import pytest

from superslm_amd.batch_ops import BatchOps, GemmLoraArgs, Lora, LogitRule, PickArgs, SharedAttentionArgs

INVALID, SMALL, MISALIGNED = 1, 2, 3
ANY = 1 << 20  # a non-null, aligned address that no refused call reads


@pytest.fixture(scope="module")
def ops(hip_lib):
    return BatchOps(hip_lib)


def test_struct_sizes():
    assert [ctypes.sizeof(t) for t in (SharedAttentionArgs, Lora, GemmLoraArgs, LogitRule, PickArgs)] == \
        [232, 40, 112, 56, 64]


def attention(ops, **change):
    f = dict(rows=3, heads=12, kv_heads=2, head_dim=128, prefixes=1, blocks=4, max_prefix=100, max_own=20, kv_pool=ANY,
             block_bytes=2 * 2 * 128 * 128, k_offset=0, v_offset=2 * 128 * 128, cap=128, q=ANY, q_scale=ANY, khead_m=ANY,
             khead_e=ANY, ln2_q=1, b_q=1, ca_q=1, ctx_fold=ANY, site=(1 << 30, 0), row_block=ANY, row_width=ANY,
             prefix_rows=ANY, prefix_block=ANY, prefix_len=ANY, codes=ANY, scales=ANY, status=ANY, workspace=ANY,
             workspace_bytes=1 << 40)
    f.update(change)
    return ops.shared_attention(**f)


@pytest.mark.parametrize("change,status", [
    ({"rows": 0}, INVALID), ({"rows": 70000}, INVALID), ({"heads": 13}, INVALID), ({"kv_heads": 0}, INVALID),
    ({"heads": 1}, INVALID), ({"head_dim": 96}, INVALID), ({"heads": 66, "head_dim": 128}, INVALID),
    ({"prefixes": -1}, INVALID), ({"prefixes": 4}, INVALID), ({"blocks": 0}, INVALID), ({"max_prefix": -1}, INVALID),
    ({"max_own": -1}, INVALID), ({"max_own": (1 << 24) + 1}, INVALID), ({"cap": 0}, INVALID), ({"cap": 129}, INVALID),
    ({"block_bytes": 2 * 2 * 128 * 128 + 8}, INVALID), ({"k_offset": 8}, INVALID), ({"v_offset": -16}, INVALID),
    ({"v_offset": 2 * 128 * 128 + 16}, INVALID), ({"kv_pool": ANY + 8}, INVALID), ({"q": ANY + 4}, INVALID),
    *[({k: None}, INVALID) for k in ("kv_pool", "q", "q_scale", "khead_m", "khead_e", "ctx_fold", "row_block", "row_width",
                                     "prefix_rows", "prefix_block", "prefix_len", "codes", "scales", "status", "workspace")],
    ({"workspace": ANY + 16}, MISALIGNED), ({"workspace_bytes": 100}, SMALL),
])
def test_attention_refusals(change, status, ops):
    assert attention(ops, **change)(raw=True) == status


def lora(ops, **change):
    f = dict(m=4, n=64, k=64, adapter_count=1, a=ANY, w=ANY, fold=ANY, in_scale=ANY, site=(1 << 30, 0), adapters=ANY,
             row_adapter=ANY, codes=ANY, scales=ANY, status=ANY, workspace=ANY, workspace_bytes=1 << 40)
    f.update(change)
    return ops.gemm_lora_requant(**f)


@pytest.mark.parametrize("change,status", [
    ({"m": 0}, INVALID), ({"m": 513}, INVALID), ({"n": 0}, INVALID), ({"n": 24}, INVALID), ({"n": 8208}, INVALID),
    ({"k": 0}, INVALID), ({"k": 24}, INVALID), ({"k": 32784}, INVALID), ({"adapter_count": -1}, INVALID),
    ({"a": ANY + 8}, INVALID), ({"w": ANY + 1}, INVALID),
    *[({k: None}, INVALID) for k in ("a", "w", "fold", "in_scale", "adapters", "row_adapter", "codes", "scales", "status",
                                     "workspace")],
    ({"workspace": ANY + 128}, MISALIGNED), ({"workspace_bytes": 10}, SMALL),
])
def test_lora_refusals(change, status, ops):
    assert lora(ops, **change)(raw=True) == status


def pick(ops, **change):
    f = dict(rows=2, vocab=100, logits=ANY, rules=ANY, tokens=ANY, adjusted=ANY, workspace=ANY, workspace_bytes=1 << 30)
    f.update(change)
    return ops.pick_tokens(**f)


@pytest.mark.parametrize("change,status", [
    ({"rows": 0}, INVALID), ({"rows": 65536}, INVALID), ({"vocab": 0}, INVALID), ({"logits_ld": 99}, INVALID),
    ({"adjusted_ld": 50}, INVALID), ({"logits": ANY + 2}, INVALID), ({"adjusted": ANY + 1}, INVALID),
    *[({k: None}, INVALID) for k in ("logits", "rules", "tokens", "workspace")],
    ({"workspace": ANY + 8}, MISALIGNED), ({"workspace_bytes": 7}, SMALL),
])
def test_pick_refusals(change, status, ops):
    assert pick(ops, **change)(raw=True) == status


def test_a_struct_of_another_size_is_refused(ops):
    for call in (attention(ops), lora(ops), pick(ops)):
        call.args.struct_size -= 8
        assert call(raw=True) == INVALID


def test_workspace_of_sizes_outside_the_domain_is_zero(ops):
    assert ops.shared_attention_workspace(0, 4, 2, 32, 0, 0, 0) == 0
    assert ops.gemm_lora_workspace(1, 8, 16) == 0
    assert ops.pick_workspace(1, 0) == 0
    assert ops.pick_workspace(1, 1) > 0 and ops.gemm_lora_workspace(1, 16, 16) > 0
    assert ops.shared_attention_workspace(1, 4, 2, 32, 0, 0, 1) > 0


def test_an_unknown_field_is_an_error(ops):
    with pytest.raises(TypeError):
        pick(ops, colour=1)
