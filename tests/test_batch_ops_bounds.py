"""Sizes at the edge of what the batch operators' launches hold (no GPU is touched)."""
import pytest

from superslm_amd.batch_ops import BatchOps
from superslm_amd.sslm import Seq

INVALID, SMALL = 1, 2
ANY = 1 << 20  # a non-null, aligned address that no refused call reads


@pytest.fixture(scope="module")
def ops(hip_lib):
    return BatchOps(hip_lib)


def attention(ops, rows, heads, kv_heads, dim, prefixes, max_prefix, max_own, workspace_bytes):
    half = kv_heads * 64 * dim
    return ops.shared_attention(rows=rows, heads=heads, kv_heads=kv_heads, head_dim=dim, prefixes=prefixes, blocks=4,
                                max_prefix=max_prefix, max_own=max_own, kv_pool=ANY, block_bytes=2 * half, k_offset=0,
                                v_offset=half, cap=64, q=ANY, q_scale=ANY, khead_m=ANY, khead_e=ANY, ln2_q=1, b_q=1, ca_q=1,
                                ctx_fold=ANY, site=(1 << 30, 0), row_block=ANY, row_width=ANY, prefix_rows=ANY,
                                prefix_block=ANY, prefix_len=ANY, codes=ANY, scales=ANY, status=ANY, workspace=ANY,
                                workspace_bytes=workspace_bytes)(raw=True)


def test_attention_grids_stay_below_two_to_the_32_threads(ops):
    """A wave of each prefix's tiles and of each row, 256 threads to four waves: 65535 rows with a prefix each over 256
    KV heads of one query head are 66558 x 256 + 65535 x 64 blocks, more than a launch takes (2^24 - 1 of them)."""
    full = (65535, 256, 256, 32, 65535, 64, 1)
    assert ops.shared_attention_workspace(*full) == 0
    assert attention(ops, *full, workspace_bytes=1 << 45) == INVALID
    # the largest ones that fit are sized, and refused here for their workspace alone
    for fits in ((50000, 256, 256, 32, 50000, 64, 1), (65535, 256, 256, 32, 1, 64, 1), (65535, 128, 128, 64, 65535, 64, 1)):
        assert ops.shared_attention_workspace(*fits) > 0
        assert attention(ops, *fits, workspace_bytes=1000) == SMALL


@pytest.mark.parametrize("rows", [1, 7, 64, 1000, 65535])
@pytest.mark.parametrize("heads,kv_heads,dim", [(1, 1, 32), (256, 256, 32), (256, 1, 32), (28, 4, 128), (32, 32, 256)])
def test_attention_workspace_holds_its_planes(rows, heads, kv_heads, dim, ops):
    """At least the int32 contexts of one plane of each kind, at every length; longer ones never need less."""
    last = 0
    for width in (1, 64, 65, 4096, 1 << 20, 1 << 24):
        n = ops.shared_attention_workspace(rows, heads, kv_heads, dim, min(rows, 3), width, width)
        assert n >= 2 * 4 * rows * heads * dim
        assert n >= last
        last = n


@pytest.mark.parametrize("field,value", [("rows", (1 << 32) + 3), ("heads", 1 << 31), ("blocks", -(1 << 31) - 1), ("cap", 1 << 63)])
def test_an_integer_past_its_field_is_an_error(field, value, ops):
    """Not the call with the integer's low bits."""
    half = 2 * 64 * 32
    f = dict(rows=3, heads=4, kv_heads=2, head_dim=32, prefixes=0, blocks=4, max_prefix=0, max_own=1, kv_pool=ANY, block_bytes=2 * half,
             k_offset=0, v_offset=half, cap=64, q=None, workspace=ANY, workspace_bytes=1 << 30, site=(1 << 30, -45))
    ops.shared_attention(**f)
    with pytest.raises(OverflowError):
        ops.shared_attention(**{**f, field: value})


@pytest.mark.parametrize("rules", [{"repetition": 32768.0}, {"repetition": 1e6}, {"presence": 1 << 31}, {"frequency": -(1 << 31) - 1},
                                   {"bias": [(3, 1 << 31)]}, {"bias": {1 << 32: 5}}])
def test_rules_past_32_bits_are_an_error(rules):
    seq = Seq.__new__(Seq)
    seq._rules = lambda ref, raw: "called"
    assert seq.set_rules(repetition=1.5, presence=-7, frequency=3, bias={4: -9}) == "called"
    with pytest.raises(OverflowError):
        seq.set_rules(**rules)
