"""Shared-prompt attention in its launches by planes, against the oracle's 64- and 128-bit arithmetic: blocks whose
rows differ in the arithmetic that they need.

Rows of up to 2 x 64 (two steps; 128 positions each where a KV head has at most 8 query heads) positions for each of
the 8 / kv_heads waves of a KV head run in one launch instead, which tests/test_gpu_batch_ops.py covers."""
import pytest

import batch_ops_ref as ref
from superslm_amd.sslm_artifact import scale_me
from test_gpu_batch_ops import Attention, dev, host, ops  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


def takes_planes(a, max_prefix=None, max_own=None):
    """The launch rule: more heads, dims or steps than the one-launch form holds."""
    g = a.nh // a.nkv
    if a.nkv > 8 or 8 % a.nkv or g > 16 or a.nh * a.d > 4096 or a.d > 128:
        return True
    step = 128 if g <= 8 else 64
    longest = (a.max_prefix if a.prefixes else 0) + a.max_own
    return -(-longest // step) > 2 * (8 // a.nkv)


def ok_rows(got):
    return int((got[2] == 0).sum())


def fast(host, a, r, kvh):  # noqa: F811
    """Whether the row's i-exp values and their sum are exact in doubles: a sum below 2^53."""
    st, c = ref.row_constants(host, a.q_scale[r].tolist(), a.khead[kvh], int(a.widths[r]))
    assert st == 0
    return (c[1] * c[1] + c[2]) * int(a.widths[r]) < 2 ** 53


@pytest.mark.parametrize("heads,kv_heads,dim,prompt", [(12, 2, 128, 1900), (28, 4, 128, 777), (8, 1, 32, 2100), (8, 2, 256, 300), (20, 1, 64, 500)])
@pytest.mark.parametrize("order", [1, -1])
def test_blocks_whose_rows_differ_in_their_arithmetic(heads, kv_heads, dim, prompt, order, ops, dev, host):  # noqa: F811
    """Rows of one prompt whose sums fit doubles beside rows whose sums do not: row by row, so that the lanes of a
    wave differ, then 10 of a kind, so that the waves of a block do; the former from peaked to flat, with sums
    of less and of more than 36 bits."""
    rows = 30
    a = Attention(heads + prompt, heads, kv_heads, dim, [(prompt, rows)], [prompt + 1 + 3 * i for i in range(rows)])
    assert takes_planes(a)
    a.khead = [scale_me(1e-4)] * kv_heads
    flat = [i % 3 == 0 if i < 10 else i < 20 for i in range(rows)][::order]
    for r in range(rows):  # a unit of score is worth 1e-4 of these
        a.q_scale[r] = scale_me(1.8e-3 if flat[r] else 100 * 10 ** (-4 * r / (rows - 1)))
    assert all(fast(host, a, r, k) != flat[r] for r in range(rows) for k in range(kv_heads))
    print(f"case planes mixed {heads}/{kv_heads}x{dim} {order}", flush=True)
    got = a.run(ops, dev)
    a.check(host, got)
    assert ok_rows(got) == rows
