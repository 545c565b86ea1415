"""The paged cache's update where its arrays are one buffer, as a decode step that keeps everything has them: a row's keep is
its length, and its new length takes that place.  The call's later reads must not see what it writes."""
import numpy as np
import pytest

import cache_ops_ref as ref
from superslm_amd.cache_ops import CacheOps
from superslm_amd.device import Device

pytestmark = pytest.mark.gpu

LEFT = 77


@pytest.fixture(scope="module")
def ops(hip_lib):
    return CacheOps(hip_lib)


@pytest.fixture(scope="module")
def dev(hip_lib):
    return Device(hip_lib)


def check(ops, dev, p, pages, tables, lengths, source, room, one, in_place):
    """keep = lengths by their numbers; `one`: which of the four arrays are one buffer."""
    rows, width = tables.shape
    rng = np.random.default_rng(1)
    pool = rng.integers(-127, 128, size=(pages, 48), dtype=np.int8)
    host = dict(lengths=lengths, keep=lengths, room=room, new_lengths=np.full(rows, LEFT, np.int64))
    shared = dev.upload(host[one[0]])
    b = {n: shared if n in one else dev.upload(x) for n, x in host.items()}
    d, t, s = dev.upload(pool), dev.upload(tables), dev.upload(source)
    new = t if in_place else dev.upload(np.full_like(tables, LEFT))
    result = dev.upload(np.full(4, LEFT, np.int32))
    n = ops.update_workspace(rows, pages, width)
    ws = dev.upload(np.full(n, 0xA5, np.uint8))
    ops.update(rows=rows, pages=pages, page_tokens=p, table_ld=width, pool=d.ptr, page_bytes=48, tables=t.ptr, source=s.ptr, new_tables=new.ptr,
               result=result.ptr, workspace=ws.ptr, workspace_bytes=n, **{k: x.ptr for k, x in b.items()})()
    assert ops.lib.lib.sslm_hip_synchronize() == 0
    want = ref.update(tables, lengths, source, lengths, room, p, pages)
    assert want[0][0] == 0 and result.numpy().tolist() == want[0]
    assert (new.numpy() == want[1]).all(), np.argwhere(new.numpy() != want[1])[:5]
    assert (b["new_lengths"].numpy() == room).all()
    for x, y in want[2]:
        pool[y] = pool[x]
    assert (d.numpy() == pool).all()


ONE = [("lengths", "keep", "new_lengths"), ("keep", "new_lengths"), ("room", "new_lengths"), ("lengths", "new_lengths")]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("one", range(len(ONE)))
@pytest.mark.parametrize("rows,width", [(1, 3), (5, 65), (37, 100), (9, 700), (150, 21)])
def test_a_step_that_keeps_everything(ops, dev, rows, width, one, in_place):
    """Tables within a wave, over several and over several blocks; rows that end at a page's border open a page."""
    p = 16
    rng = np.random.default_rng(rows)
    held = rng.integers(0, width - 1, rows)  # whole pages of a row
    lengths = held * p + np.where(np.arange(rows) % 3 == 1, rng.integers(0, p, rows), 0)
    need = -(-lengths // p)
    pages = int(need.sum()) + 2 * rows + 3
    order, at = rng.permutation(pages), 0
    tables = np.full((rows, width), -1, np.int32)
    for r, m in enumerate(need):
        tables[r, :m] = order[at:at + m]
        at += m
    room = np.minimum(lengths + rng.integers(1, 2 * p, rows), width * p)
    source = np.where(lengths > 0, np.arange(rows), -1).astype(np.int32)
    check(ops, dev, p, pages, tables, lengths, source, room, ONE[one], in_place)


def test_forks_of_equal_length(ops, dev):
    """Four answers to each of six prompts: the open page is copied, the next ones are new."""
    rows, width, p = 24, 90, 16
    for length in (80 * p, 80 * p + 5):
        lengths, tables = np.full(rows, length, np.int64), np.full((rows, width), -1, np.int32)
        for r in range(rows):
            tables[r, :81] = np.arange(81) + 81 * (r // 4)
        source = (np.arange(rows) // 4 * 4).astype(np.int32)
        check(ops, dev, p, 81 * 6 + 100, tables, lengths, source, lengths + 1 + np.arange(rows), ONE[0], True)


@pytest.mark.parametrize("in_place", [False, True])
def test_a_table_of_several_sweeps(ops, dev, in_place):
    """A table of more entries than a launch has threads: the thread that writes the row's new length comes to its new page afterwards."""
    p, whole = 16, 2048 * 256
    lengths, width = np.array([whole * p], np.int64), whole + 8
    tables = np.full((1, width), -1, np.int32)
    tables[0, :whole] = np.arange(whole) % 11
    check(ops, dev, p, 14, tables, lengths, np.zeros(1, np.int32), lengths + 20, ONE[0], in_place)
