"""Shared-prompt attention in its launches by planes, against the oracle's 64- and 128-bit arithmetic: prompts whose
query rows fill several blocks, every softmax scale, blocks whose rows differ in the arithmetic that they need,
refusals; and the planes' workspace on streams and in graphs.

Rows of up to 2 x 64 (two steps; 128 positions each where a KV head has at most 8 query heads) positions for each of
the 8 / kv_heads waves of a KV head run in one launch instead, which tests/test_gpu_batch_ops.py covers."""
import os
import shutil
import subprocess

import numpy as np
import pytest

import batch_ops_ref as ref
from conftest import HIP_SO, ROOT
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


@pytest.mark.parametrize("heads,kv_heads,dim,runs,loose", [
    # a block holds 64 query rows of one prefix and KV head: 23 x 6 = 138 (the last block 10, in one tile), 13 x 6 = 78
    (12, 2, 128, [(1531, 23), (900, 13)], [40, 1600]),
    # 7 heads to a KV head: 21 x 7 = 147, 10 x 7 = 70, an empty run between, one row of 7
    (28, 4, 128, [(700, 21), (65, 0), (333, 10), (64, 1)], [513]),
    # exactly one block and exactly two, then a single row more
    (8, 1, 32, [(2100, 8), (2049, 16), (130, 17)], []),
    # 20 heads to a KV head (tiles that hold parts of two rows), a prefix of several blocks per row count
    (20, 1, 64, [(200, 10), (130, 33)], [1, 0]),
    # one head to a KV head, 16 rows to a tile
    (16, 16, 64, [(300, 70)], [12]),
    # head size 256
    (8, 2, 256, [(150, 17), (70, 36)], [90]),
])
def test_prompts_of_several_blocks(heads, kv_heads, dim, runs, loose, ops, dev, host):  # noqa: F811
    rng = np.random.default_rng(heads + dim)
    widths = [n + int(rng.integers(0, 70)) for n, rows in runs for _ in range(rows)] + loose
    widths[1] = max(1, widths[1] - runs[0][0] // 2)  # one row ends inside its prompt
    a = Attention(sum(widths) + dim, heads, kv_heads, dim, runs, widths)
    assert takes_planes(a) and max(rows * heads // kv_heads for _, rows in runs) > 64
    print(f"case planes {heads}/{kv_heads}x{dim} {runs}", flush=True)
    a.check(host, a.run(ops, dev))


@pytest.mark.parametrize("scale", [1e-2, 3e-4, 2e-5, 1e-6, 5e-7, 3e-7, 1.6e-7])
def test_planes_over_the_softmax_scales(scale, ops, dev, host):  # noqa: F811
    """From peaked rows to flat ones whose i-exp values and sums pass 32 and 52 bits; at the last scale some rows are
    past the softmax's own gate and are refused."""
    a = Attention(11, 12, 2, 128, [(1900, 7)], [1900, 1917, 1964, 2027, 90, 1901, 2000, 1300], scale=scale)
    assert takes_planes(a)
    print(f"case planes scale {scale}", flush=True)
    got = a.run(ops, dev)
    a.check(host, got)
    assert 0 < ok_rows(got) and (ok_rows(got) == a.rows) == (scale > 2e-7)


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


def test_planes_refuse_rows_by_their_status(ops, dev, host):  # noqa: F811
    """Each refusal in a batch by planes, beside rows of the same tile and block that are computed."""
    widths = [1901 + i for i in range(20)] + [1600 + i for i in range(12)] + [50, 60, 70]
    a = Attention(9, 12, 2, 128, [(1900, 20), (1600, 12)], widths)
    a.q_scale[1] = 1 << 30, 300     # no constant of the i-exp is left: refused in the softmax
    a.q_scale[4] = 1 << 31, -40     # outside the mantissa's domain
    a.q_scale[5] = 1 << 30, -70     # the constants cannot be derived
    a.q_scale[21] = 1 << 30, 300
    a.q_scale[22] = scale_me(5e-6)  # past the softmax's gate
    a.row_block[7] = a.blocks
    a.widths[30] = a.cap + 5
    a.widths[33] = 0
    assert takes_planes(a)
    print("case planes refusals", flush=True)
    got = a.run(ops, dev, max_own=71)
    assert [got[2][r] for r in (1, 4, 5, 21, 22, 33)] == [ref.REFUSED, ref.SCALE_MANTISSA, ref.SCALE_DERIVATION, ref.REFUSED, ref.ROW_WIDTH,
                                                          ref.ROW_WIDTH]
    a.check(host, got, expect={7: ref.POSITION_OVER_CAP, 30: ref.POSITION_OVER_CAP})
    assert ok_rows(got) == a.rows - 8
    a.prefix_block[1] = -1  # a prompt of no block: its rows alone
    got = a.run(ops, dev, max_own=71)
    a.check(host, got, rows=range(20), expect={7: ref.POSITION_OVER_CAP})
    assert (got[2][20:32] == ref.POSITION_OVER_CAP).all() and got[2][34] == 0


def test_planes_with_looser_maxima(ops, dev, host):  # noqa: F811
    a = Attention(7, 12, 2, 128, [(1100, 14), (51, 3)], [1100 + 5 * i for i in range(14)] + [60, 51, 52] + [20])
    assert takes_planes(a)
    want = a.run(ops, dev)
    a.check(host, want)
    for more in (1, 500, 70000):
        print(f"case planes maxima +{more}", flush=True)
        got = a.run(ops, dev, max_prefix=a.max_prefix + more, max_own=a.max_own + more)
        assert all(np.array_equal(x, y) for x, y in zip(got, want))


def test_planes_on_streams_and_in_graph_replays(tmp_path):
    """Two batches by planes at once, each with its own workspace: on two streams, as two captured graphs, as the
    branches of one, over new inputs (tests/batch_ops_planes_graph_check.cpp, built here)."""
    if shutil.which("hipcc") is None:
        pytest.skip("hipcc not available")
    obj, exe = str(tmp_path / "check.o"), str(tmp_path / "batch_ops_planes_graph_check")
    subprocess.run(["hipcc", "-O1", "-std=c++17", "-w", "--offload-arch=gfx950", "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", "-c", os.path.join(ROOT, "tests", "batch_ops_planes_graph_check.cpp"), "-o", obj], check=True)
    libdir = os.path.dirname(HIP_SO)
    subprocess.run(["hipcc", obj, "-L" + libdir, "-lsslm_hip", "-Wl,-rpath," + libdir, "-o", exe], check=True)
    print("case planes on streams and in graphs", flush=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.strip().splitlines()[-1].startswith("ok"), (r.returncode, r.stdout, r.stderr[-2000:])
