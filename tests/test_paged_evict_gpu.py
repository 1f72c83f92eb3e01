"""Eviction on the GPU, in 16 bits and in 4: which tokens stay, where they and their masses go, lengths and free pages, against
Python integers (paged4check.ref_evict). Everything is compared bit by bit, what must not change among it."""

import numpy as np
import pytest

import notcute_flash as nc
import paged4check as p4
from pagedcheck import Pool, make_table

pytestmark = pytest.mark.gpu


def _masses(rng, R, room, kind):
    if kind == "ties":
        return rng.integers(0, 4, (R, room)).astype(np.float32)
    if kind == "zeros":
        return np.where(rng.random((R, room)) < 0.5, 0.0, -0.0).astype(np.float32)
    if kind == "odd":  # infinities, NaN of both signs, negative and subnormal numbers, both zeros
        pick = np.array([np.inf, -np.inf, np.nan, 1.0, -1.0, 1e-42, -1e-42, 0.0, -0.0, 3e38], np.float32)
        x = pick[rng.integers(0, len(pick), (R, room))]
        return np.where((rng.random((R, room)) < 0.05) & np.isnan(x), np.copysign(x, np.float32(-1)), x).astype(np.float32)
    if kind == "close":  # differ in the lowest bits only
        return (np.float32(1.0).view(np.uint32) + rng.integers(0, 300, (R, room)).astype(np.uint32)).view(np.float32)
    return np.exp(2 * rng.standard_normal((R, room))).astype(np.float32)


def _evict(gpu, pool, four, table, lens, mass, free, cursor, rules, in_place=False, mass_stride=0, stream=None):
    R = len(lens)
    o = nc.paged_options(num_seqs=R, max_pages=table.shape[1], num_q_heads=pool.heads, **pool.options())
    bufs = pool.upload()
    dt, dl, dm, df = (nc.DeviceBuffer.from_array(x) for x in (table, lens, mass, free))
    dc = nc.DeviceBuffer.from_array(np.array([cursor, -7, -7, -7], np.int32))
    kept = dl if in_place else nc.DeviceBuffer.from_array(np.full(R + 1, -7, np.int32))
    counts = dc if in_place else nc.DeviceBuffer(16)
    work = nc.DeviceBuffer(nc.paged_evict_workspace_bytes(o))
    work.memset(0xAB)
    f = nc.paged4_evict if four else nc.paged_evict
    f(gpu, dt, dl, dm, *bufs, df, p4.View(dc, 0, 4), kept, counts, work, nc.evict_rules(**dict(zip(("limit", "budget", "sinks", "recent"), rules))), o,
      stream, mass_stride=mass_stride)
    nc.synchronize()
    assert np.array_equal(dt.download(np.int32, table.size), table.ravel())
    if not in_place:
        assert np.array_equal(dl.download(np.int32, R), lens) and kept.download(np.int32, R + 1)[R] == -7
    data = pool.download(*bufs) if not four else sum(pool.download(bufs), [])
    return data, kept.download(np.int32, R), dm.download(np.float32, mass.size).reshape(mass.shape), df.download(np.int32, free.size), counts.download(
        np.int32, 4)


def _move(pool, four, table, kept):
    """Moves the pool's rows as the lists say."""
    for r, keep in enumerate(kept):
        if keep is None:
            continue
        ps, heads = pool.ps, np.arange(pool.heads)[None, :]
        rows = [(table[r, j // ps], j % ps) for j in keep]
        page, tok = (np.array(x)[:, None] for x in zip(*rows))
        to = [(table[r, j // ps], j % ps) for j in range(len(keep))]
        tp, tt = (np.array(x)[:, None] for x in zip(*to))
        here = ((page >= 0) & (page < pool.pages) & (tp >= 0) & (tp < pool.pages))[:, 0]
        page, tok, tp, tt = page[here], tok[here], tp[here], tt[here]
        for which in range(2):
            if four:
                at, d = pool._at(page, heads, tok) + which * pool.gap, pool.d
                i = 0 if pool.gap else which
                codes = pool.codes[i][at[..., None] + np.arange(d)]
                pool.put(which, tp, heads, tt, codes, pool.scales[i][at[..., None] // 32 + np.arange(d // 32)])
            else:
                pool.put(which, tp, heads, tt, pool.get(which, page, heads, tok))


CASES = [  # lens, limit, budget, sinks, recent, masses, four, heads, d, page size, layout
    ([10], 5, 3, 0, 0, "exp", False, 1, 16, 16, "hnd"), ([10, 4, 0, 9], 4, 4, 1, 1, "exp", False, 2, 64, 4, "nhd"),
    ([10, 4, 5, 9], 4, 4, 1, 1, "ties", True, 2, 64, 4, "hnd"), ([300, 257, 256, 1], 256, 128, 4, 64, "exp", True, 3, 32, 16, "nhd"),
    ([300] * 5, 256, 1, 0, 0, "ties", False, 1, 128, 7, "hnd"), ([300] * 5, 256, 1, 1, 0, "exp", False, 1, 32, 7, "inter"),
    ([300] * 3, 256, 1, 0, 1, "exp", True, 1, 128, 1, "inter"), ([500, 100], 200, 200, 100, 100, "exp", False, 2, 64, 16, "hnd"),
    ([1500, 1025, 1024], 1000, 999, 0, 0, "zeros", False, 1, 16, 24, "nhd"), ([2000, 3000], 1500, 700, 3, 100, "odd", True, 2, 64, 16, "hnd"),
    ([2000, 1800], 1500, 700, 3, 100, "close", False, 1, 32, 100, "hnd"), ([9000, 8193, 8192], 8192, 4000, 16, 500, "exp", False, 1, 64, 16, "hnd"),
    ([20000, 30, 12345], 5000, 5000, 4, 1000, "ties", True, 1, 32, 16, "nhd"), ([17000], 16384, 16000, 0, 0, "close", False, 1, 16, 64, "hnd"),
    ([40] * 1100, 39, 20, 2, 5, "exp", False, 1, 16, 16, "hnd"), ([0, 0, 0], 5, 5, 0, 0, "exp", False, 1, 16, 16, "hnd"),
    ([12000], 2, 1, 0, 0, "odd", False, 1, 16, 16, "hnd"), ([700, 650, 3], 600, 599, 0, 0, "exp", True, 5, 128, 16, "nhd"),
    # rows moved by several workgroups each: by one place, most of them, with others' heads, chains in turn, chunks in turn
    ([3000, 5, 2999], 2998, 2998, 0, 0, "zeros", False, 2, 128, 16, "hnd"), ([6000, 5999], 5999, 5998, 1, 0, "exp", True, 3, 128, 7, "nhd"),
    ([3000, 1700], 1699, 1000, 0, 900, "exp", False, 4, 32, 16, "nhd"), ([5000], 4000, 3000, 8, 8, "ties", True, 8, 32, 16, "nhd"),
    ([5000, 4100], 4000, 3900, 8, 8, "exp", True, 6, 64, 16, "nhd"), ([4000], 3999, 3998, 0, 0, "exp", False, 12, 16, 5, "nhd"),
    ([1300] * 150, 1299, 1200, 0, 10, "exp", False, 8, 16, 16, "hnd"), ([1000], 990, 950, 3, 10, "exp", False, 300, 128, 16, "nhd"),
    # selected from by several workgroups: nothing to choose, parts of more than a sweep, the edge in each of the passes, empty parts
    ([13000, 12300, 10], 8000, 5000, 2000, 3000, "exp", False, 1, 16, 64, "hnd"), ([140001, 70000], 60000, 50000, 7, 100, "close", False, 1, 16, 64, "hnd"),
    ([140001], 60000, 59999, 0, 0, "zeros", False, 1, 16, 64, "hnd"), ([30000, 9000, 2049], 2048, 2047, 2047, 0, "odd", False, 1, 16, 24, "nhd"),
    ([16384, 8193, 100], 4000, 2100, 2050, 1, "odd", True, 1, 32, 16, "hnd"), ([12288, 4096, 4097], 4095, 2000, 0, 1999, "ties", False, 1, 16, 16, "hnd"),
]


@pytest.mark.parametrize("lens,limit,budget,sinks,recent,kind,four,heads,d,ps,layout", CASES)
@pytest.mark.parametrize("in_place", [False, True])
def test_evict_matches_the_definition(gpu, lens, limit, budget, sinks, recent, kind, four, heads, d, ps, layout, in_place):
    rng = np.random.default_rng(sum(lens) + budget)
    lens = np.array(lens, np.int32)
    R, width = len(lens), -(-int(max(lens.max(), 1)) // ps) + 1
    held = int(sum(-(-n // ps) for n in lens))
    pages = held + 3
    pool = p4.Pool4(rng, pages, heads, ps, d, layout=layout) if four else Pool(rng, pages, heads, ps, d, layout=layout)
    table = make_table(rng, lens, ps, pages, width)
    stride = width * ps + 1
    mass = _masses(rng, R, stride, kind)
    free = rng.integers(0, 1000, pages).astype(np.int32)
    rules = (limit, budget, sinks, recent)
    kept, out, m, f, counts = p4.ref_evict(lens, mass, table, free, held, ps, width * ps, rules)
    got = _evict(gpu, pool, four, table, lens, mass, free, held, rules, in_place, stride)
    assert got[1].tolist() == out.tolist()
    assert np.array_equal(got[4], counts) and np.array_equal(got[3], f)
    assert np.array_equal(got[2].view(np.uint32), m.view(np.uint32))
    _move(pool, four, table, kept)
    for have, want in zip(got[0], pool.codes + pool.scales if four else pool.bufs):
        assert np.array_equal(have, want)


def test_lists_without_room_absent_pages_and_long_lengths(gpu):
    """A cursor that leaves no room, or stands behind the list; pages outside the pool; lengths past the table's row, and negative ones."""
    rng = np.random.default_rng(8)
    ps, width = 4, 10
    lens = np.array([1000, -3, 30, 40], np.int32)  # the first is cut to 40
    for cursor, size in ((5, 40), (0, 40), (-2, 40), (50, 40), (30, 12), (44, 43)):
        pool = Pool(rng, 40, 2, ps, 32)
        table = make_table(rng, np.array([40, 0, 30, 40]), ps, 40, width)
        table[2, 0], table[2, 3], table[3, 1], table[3, 9] = -1, 40, 2 ** 31 - 1, -(2 ** 31)
        mass = _masses(rng, 4, width * ps, "exp")
        free = np.arange(500, 500 + size, dtype=np.int32)
        rules = (20, 11, 2, 3)
        kept, out, m, f, counts = p4.ref_evict(lens, mass, table, free, cursor, ps, 40, rules)
        got = _evict(gpu, pool, False, table, lens, mass, free, cursor, rules)
        assert out.tolist() == [11, 0, 11, 11] == got[1].tolist()
        assert np.array_equal(got[3], f) and np.array_equal(got[4], counts) and np.array_equal(got[2], m)
        _move(pool, False, table, kept)
        for have, want in zip(got[0], pool.bufs):
            assert np.array_equal(have, want)


def test_no_list_at_all(gpu):
    rng = np.random.default_rng(2)
    pool = Pool(rng, 4, 1, 4, 16)
    table, mass = np.arange(4, dtype=np.int32)[None], _masses(rng, 1, 16, "exp")
    got = _evict(gpu, pool, False, table, np.array([16], np.int32), mass, np.zeros(0, np.int32), 3, (8, 4, 0, 0))
    assert got[1].tolist() == [4] and got[4].tolist() == [0, 1, 3, 12]
