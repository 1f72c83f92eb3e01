"""An eviction whose move does not see other workgroups' flags: it says so in counts[1], and moves none of the rows that it could not be sure
of. The library's own limit of tries stands in for a workspace that another call has changed: with none, every wait gives up."""

import ctypes

import numpy as np
import pytest

import notcute_flash as nc
from pagedcheck import Pool, make_table
import paged4check as p4

pytestmark = pytest.mark.gpu


@pytest.fixture
def tries():
    limit = ctypes.c_uint32.in_dll(nc.load_library(), "nc_internal_evict_tries")
    old = limit.value
    yield limit
    limit.value = old


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,chunks", [(3000, True), (13000, True), (60, False)])
def test_a_wait_that_gives_up_is_told(gpu, tries, four, in_place, n, chunks):
    """chunks: whether a head's rows are several workgroups'; where one has them all, nothing waits."""
    assert tries.value >= 1 << 16
    rng = np.random.default_rng(n)
    ps, heads, d = 16, 1, 128
    pages = -(-n // ps) + 5
    lens = np.array([n, 7], np.int32)
    pool = (p4.Pool4 if four else Pool)(rng, pages, heads, ps, d)
    table = make_table(rng, lens, ps, pages, pages)
    mass = rng.random((2, pages * ps)).astype(np.float32)
    rules = nc.evict_rules(limit=n // 2, budget=n // 2, sinks=1, recent=1)
    o = nc.paged_options(num_seqs=2, max_pages=pages, num_q_heads=heads, **pool.options())
    seen = []
    for limit in (tries.value, 0, tries.value):
        tries.value = limit
        bufs = pool.upload()
        dt, dl, dm, df = (nc.DeviceBuffer.from_array(x) for x in (table, lens, mass, np.arange(pages, dtype=np.int32)))
        dc = nc.DeviceBuffer.from_array(np.array([pages, -7, -7, -7], np.int32))
        kept, counts = (dl, dc) if in_place else (nc.DeviceBuffer(8), nc.DeviceBuffer(16))
        work = nc.DeviceBuffer(nc.paged_evict_workspace_bytes(o))
        work.memset(0xAB)
        (nc.paged4_evict if four else nc.paged_evict)(gpu, dt, dl, dm, *bufs, df, p4.View(dc, 0, 4), kept, counts, work, rules, o)
        nc.synchronize()
        data = sum(pool.download(bufs), []) if four else pool.download(*bufs)
        seen.append((counts.download(np.int32, 4).tolist(), kept.download(np.int32, 2).tolist(), data))
    freed = -(-n // ps) - -(-(n // 2) // ps)
    want = [pages - freed, 1, freed, n - n // 2]
    assert seen[0][0] == seen[2][0] == want and seen[0][1] == seen[1][1] == [n // 2, 7]
    assert seen[1][0] == ([want[0], -1, *want[2:]] if chunks else want)
    for x, y in zip(seen[0][2], seen[2][2]):
        assert np.array_equal(x, y)
    if not chunks:
        return
    # the first chunk of a head moves; what the others would have taken stands where it was
    for have, was, full in zip(seen[1][2], pool.codes + pool.scales if four else pool.bufs, seen[0][2]):
        assert ((have == was) | (have == full)).all() and not np.array_equal(have, full)
