"""The 4-bit paged cache on the GPU through the C ABI: rows in and out, and single-token attention, against the definitions in
float64 (paged4check.py)."""

import numpy as np
import pytest

import notcute_flash as nc
import paged4check as p4
from pagedcheck import SENTINEL, encode, make_table

pytestmark = pytest.mark.gpu


def _rows(rng, n, heads, d, dtype, kind="normal"):
    x = rng.standard_normal((n, heads, d))
    if kind == "wide":  # magnitudes over the type's whole range, group by group and value by value
        lo, hi = (-24, 15) if dtype == "f16" else (-130, 127)
        x = x * 2.0 ** rng.integers(lo, hi, (n, heads, d // 32)).repeat(32, axis=-1) * 2.0 ** rng.integers(-4, 1, x.shape)
        if dtype == "f16":
            x = np.clip(x, -65504, 65504)
    elif kind == "ties":  # halfway between two codes, of several scales
        x = rng.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 0.0, -0.0, 7.0], x.shape) * rng.choice([-1, 1], x.shape)
        x = x * 2.0 ** rng.integers(-8, 8, (n, heads, d // 32)).repeat(32, axis=-1)
    return encode(np.clip(x, -3.3e38, 3.3e38), dtype)


def _append(gpu, pool, bufs, k, v, slots, row_stride=0, row_head_stride=0, offset=0, stream=None):
    o = nc.paged_options(num_q_heads=pool.heads, row_stride=row_stride, row_head_stride=row_head_stride, **pool.options())
    dk, dv = nc.DeviceBuffer.from_array(k), nc.DeviceBuffer.from_array(v)
    ds = nc.DeviceBuffer.from_array(np.asarray(slots, np.int32))
    nc.paged4_append(gpu, p4.View(dk, 2 * offset), p4.View(dv, 2 * offset), ds, *bufs, o, stream)
    nc.synchronize()


CASES = [  # rows, heads, d, page size, layout, pad, type, kind, row pad, offset
    (1, 1, 32, 16, "hnd", 0, "f16", "normal", 0, 0), (5, 2, 64, 7, "nhd", 0, "bf16", "normal", 0, 0),
    (33, 3, 128, 16, "hnd", 32, "f16", "normal", 3, 1), (200, 8, 64, 24, "inter", 0, "bf16", "normal", 0, 0),
    (64, 2, 32, 1, "inter", 32, "f16", "wide", 1, 3), (64, 5, 64, 16, "nhd", 0, "bf16", "wide", 0, 0), (40, 1, 128, 100, "hnd", 0, "f16", "wide", 0, 0),
    (50, 2, 64, 16, "hnd", 0, "f16", "ties", 0, 0), (50, 2, 64, 16, "hnd", 0, "bf16", "ties", 5, 1),
]


@pytest.mark.parametrize("n,heads,d,ps,layout,pad,dtype,kind,row_pad,offset", CASES)
def test_append_and_read_are_exact(gpu, n, heads, d, ps, layout, pad, dtype, kind, row_pad, offset):
    rng = np.random.default_rng(n + d)
    pages = -(-n // ps) + 2
    pool = p4.Pool4(rng, pages, heads, ps, d, dtype, layout, pad)
    bufs = pool.upload()
    slots = rng.permutation(pages * ps)[:n].astype(np.int32)
    slots[n // 2] = -1 if n > 1 else slots[0]
    if n > 8:
        slots[3] = pages * ps  # behind the pool
    wide = heads * d + row_pad
    raw = []
    for which in range(2):
        x = _rows(rng, n, heads, d, dtype, kind)
        buf = np.full(n * wide + offset, 0x7E00, np.uint16)
        for i in range(n):
            buf[offset + i * wide:offset + i * wide + heads * d] = x[i].ravel()
        raw.append((x, buf))
    _append(gpu, pool, bufs, raw[0][1], raw[1][1], slots, row_stride=wide, offset=offset)
    ok = [i for i in range(n) if 0 <= slots[i] < pages * ps]
    for which in range(2):
        x = p4.decode_bits(raw[which][0], dtype)
        for i in ok:
            pool.put_values(which, slots[i] // ps, np.arange(heads), slots[i] % ps, x[i])
    codes, scales = pool.download(bufs)
    for have, want in zip(codes + scales, pool.codes + pool.scales):
        assert np.array_equal(have, want)
    # back again, some rows twice, to rows of another pitch
    again = np.concatenate([slots, slots[:2]])
    out_wide = heads * d + 3
    o = nc.paged_options(num_q_heads=heads, row_stride=out_wide, **pool.options())
    size = len(again) * out_wide + 1
    dk, dv = (nc.DeviceBuffer.from_array(np.full(size, 0x1234, np.uint16)) for _ in range(2))
    nc.paged4_read(gpu, *bufs, nc.DeviceBuffer.from_array(again), p4.View(dk, 2), p4.View(dv, 2), o)
    nc.synchronize()
    for which, b in enumerate((dk, dv)):
        got = b.download(np.uint16, size)
        want = np.full(size, 0x1234, np.uint16)
        for i, s in enumerate(again):
            x = np.zeros((heads, d)) if not 0 <= s < pages * ps else pool.get(which, s // ps, np.arange(heads), s % ps)
            want[1 + i * out_wide:1 + i * out_wide + heads * d] = encode(x, dtype).ravel()
        g, w = (p4.decode_bits(x, dtype) for x in (got, want))
        assert np.array_equal(g, w) and np.array_equal(np.signbit(g), np.signbit(w))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_append_marks_groups_that_are_not_finite(gpu, dtype):
    pool = p4.Pool4(np.random.default_rng(1), 3, 2, 16, 64, dtype)
    bufs = pool.upload()
    x = np.random.default_rng(2).standard_normal((3, 2, 64))
    x[0, 1, 40], x[1, 0, 3], x[2, 1, 63] = np.nan, np.inf, -np.inf
    bits = encode(x, dtype)
    _append(gpu, pool, bufs, bits, bits, [5, 17, 47])
    for which in range(2):
        for i, s in enumerate((5, 17, 47)):
            pool.put_values(which, s // 16, np.arange(2), s % 16, p4.decode_bits(bits[i], dtype))
    codes, scales = pool.download(bufs)
    for have, want in zip(codes + scales, pool.codes + pool.scales):
        assert np.array_equal(have, want)
    assert sum(int((s == 255).sum()) for s in scales) == 6


def _decode(gpu, pool, q, table, lens, mass=None, mass_stride=0, q_off=0, q_pad=0, o_pad=0, stream=None, work=None, scale=None):
    """(o, mass) of one call, with sentinels around O and behind the last request."""
    R, Hq, d = q.shape
    opts = nc.paged_options(num_seqs=R, num_q_heads=Hq, max_pages=table.shape[1], q_head_stride=d + q_pad, o_head_stride=d + o_pad, scale=scale,
                            **pool.options())
    qb = np.zeros((R, Hq, d + q_pad), np.uint16)
    qb[:, :, :d] = q
    dq = nc.DeviceBuffer.from_array(np.concatenate([np.zeros(q_off, np.uint16), qb.ravel()]))
    out = np.full((R + 1) * Hq * (d + o_pad), SENTINEL, np.float32)
    do, dt, dl = (nc.DeviceBuffer.from_array(x) for x in (out, table, np.asarray(lens, np.int32)))
    bufs = pool.upload()
    dm = None if mass is None else nc.DeviceBuffer.from_array(mass)
    if work is None:
        work = nc.DeviceBuffer(nc.paged4_workspace_bytes(opts, mass is not None))
        work.memset(0)
    nc.paged4_decode(gpu, p4.View(dq, 2 * q_off), *bufs, dt, dl, do, work, opts, stream, mass=dm, mass_stride=mass_stride)
    nc.synchronize()
    o = do.download(np.float32, out.size).reshape(R + 1, Hq, d + o_pad)
    assert (o[R] == SENTINEL).all() and (o[:, :, d:] == SENTINEL).all()
    assert not work.download(np.uint32, 5 * 2 * 1024).any()  # the counters are as they were
    return o[:R, :, :d], None if mass is None else dm.download(np.float32, mass.size).reshape(mass.shape)


def _q(rng, R, Hq, d, dtype, sigma=1.0):
    return encode(sigma * rng.standard_normal((R, Hq, d)), dtype)


SHAPES = [  # lens, kv heads, group, d, page size, layout, type
    ([1], 1, 1, 32, 16, "hnd", "f16"), ([1, 2, 16], 2, 4, 64, 16, "hnd", "bf16"), ([17, 0, 63, 64, 65], 2, 4, 128, 16, "hnd", "f16"),
    ([100, 257, 31], 3, 5, 64, 32, "nhd", "bf16"), ([300, 0, 1, 129], 4, 1, 32, 16, "inter", "f16"), ([77, 513], 1, 16, 128, 48, "nhd", "bf16"),
    ([5, 700, 33], 2, 3, 64, 7, "hnd", "f16"), ([1000, 3], 2, 8, 128, 24, "nhd", "bf16"), ([40, 41, 42], 2, 4, 32, 1, "inter", "bf16"),
    ([2100, 900], 1, 17, 64, 16, "hnd", "f16"), ([1500], 2, 40, 128, 16, "nhd", "f16"), ([600, 70], 1, 70, 32, 100, "hnd", "bf16"),
    ([3000], 4, 4, 64, 16, "nhd", "bf16"), ([3000, 2000], 8, 2, 32, 5, "nhd", "f16"), ([513, 514], 4, 2, 128, 16, "nhd", "f16"),
    ([60] * 90, 8, 2, 64, 16, "hnd", "f16"), ([20] * 300, 8, 1, 32, 7, "hnd", "bf16"), ([30, 0] * 100, 8, 4, 128, 16, "nhd", "bf16"),
    ([12000], 1, 4, 128, 64, "hnd", "f16"), ([700, 3, 1200], 4, 3, 128, 1, "hnd", "f16"), ([900], 6, 4, 128, 1, "nhd", "bf16"),
    ([800, 100], 4, 8, 64, 1, "nhd", "f16"), ([600, 530, 1, 0, 700] * 2, 4, 3, 128, 24, "nhd", "f16"), ([515] * 40, 2, 1, 128, 7, "nhd", "bf16"),
    ([700, 3, 1200] * 3, 6, 4, 128, 1, "hnd", "f16"), ([7300, 7600, 600] * 8, 8, 7, 32, 16, "nhd", "f16"),
    ([15000, 0, 14000, 9] * 2, 8, 8, 64, 16, "nhd", "bf16"), ([14900] * 8, 4, 5, 128, 40, "nhd", "f16"),
]


@pytest.mark.parametrize("lens,heads,group,d,ps,layout,dtype", SHAPES)
def test_decode_matches_float64(gpu, lens, heads, group, d, ps, layout, dtype):
    rng = np.random.default_rng(len(lens) + d + ps)
    width = -(-max(lens) // ps) + 1
    pages = sum(-(-n // ps) for n in lens) + 1
    pool = p4.Pool4(rng, pages, heads, ps, d, dtype, layout, pad=32 if layout == "inter" else 0)
    table = make_table(rng, lens, ps, pages, width)
    q = _q(rng, len(lens), heads * group, d, dtype)
    want, bound, _, _ = p4.ref_attention(q, pool, table, lens, 1 / np.sqrt(d), group, True)
    got, _ = _decode(gpu, pool, q, table, lens)
    assert (np.abs(got - want) <= bound).all(), np.max(np.abs(got - want) / bound)


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("ps", [16, 9])
def test_decode_without_the_other_parts_of_memory(gpu, d, ps):
    """Odd offsets and strides of Q and O; NaN groups everywhere but in the keys that count; absent pages; negative and long lengths."""
    rng = np.random.default_rng(d + ps)
    lens = [70, -5, 3 * ps, 10 ** 6, 2 * ps + 3]
    width, pages, heads, group = 9, 60, 2, 3
    pool = p4.Pool4(rng, pages, heads, ps, d, "f16", poison=True)
    cut = [min(max(n, 0), width * ps) for n in lens]
    table = make_table(rng, cut, ps, pages, width)
    table[2, 1], table[4, 0], table[4, 1], table[4, 2] = pages, -1, 2 ** 31 - 1, -(2 ** 31)  # one absent page, all absent pages
    for r, n in enumerate(cut):
        for j in range(n):
            page = int(table[r, j // ps])
            if 0 <= page < pages:
                for which in range(2):
                    pool.put_values(which, page, np.arange(heads), j % ps, rng.standard_normal((heads, d)))
    q = _q(rng, 5, heads * group, d, "f16")
    want, bound, madd, mbound = p4.ref_attention(q, pool, table, cut, 1 / np.sqrt(d), group, True)
    mass = rng.random((5, width * ps)).astype(np.float32)
    for kw in (dict(), dict(q_off=1, q_pad=1), dict(q_off=3, o_pad=1), dict(q_pad=8, o_pad=4)):
        got, _ = _decode(gpu, pool, q, table, lens, **kw)
        assert (np.abs(got - want) <= bound).all() and not got[1].any() and not got[4].any()
        got, m = _decode(gpu, pool, q, table, lens, mass=mass, **kw)
        assert (np.abs(got - want) <= bound).all()
        assert (np.abs(m - (mass.astype(float) + madd)) <= mbound + 2.0 ** -23 * m).all()
        assert np.array_equal(m[1], mass[1]) and np.array_equal(m[4], mass[4])


@pytest.mark.parametrize("d", [32, 64, 128])
def test_decode_nan_and_infinite_inputs(gpu, d):
    """A NaN group of K or of V that counts, a query that is not finite, and one of zeros."""
    rng = np.random.default_rng(d)
    pool = p4.Pool4(rng, 8, 1, 16, d, "f16")
    table = np.arange(8, dtype=np.int32).reshape(4, 2)
    lens = [20, 20, 20, 20]
    k, v = rng.standard_normal((2, d))
    k[3], v[d - 1] = np.nan, np.inf
    pool.put_values(0, 0, 0, 5, k)
    pool.put_values(1, 2, 0, 7, v)
    q = _q(rng, 4, 2, d, "f16")
    q[2, 0, 1] = encode(np.array([np.inf]), "f16")[0]
    q[3] = 0
    got, _ = _decode(gpu, pool, q, table, lens)
    assert np.isnan(got[0]).all() and np.isnan(got[1, :, d - 32:]).all() and np.isfinite(got[1, :, :d - 32]).all()
    assert np.isnan(got[2, 0]).all() and np.isfinite(got[2, 1]).all()
    vals, _ = p4.rows_of(pool, table, lens, 3, 1, 0)
    assert np.allclose(got[3], vals.mean(0), atol=1e-5)


@pytest.mark.parametrize("dtype,spread", [("f16", 10), ("bf16", 30)])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_decode_of_far_apart_scales(gpu, d, dtype, spread):
    """Groups of K and V of very different scales, and queries whose values are."""
    rng = np.random.default_rng(d + spread)
    lens, heads, group, ps = [150, 33], 2, 4, 16
    pool = p4.Pool4(rng, 20, heads, ps, d, dtype)
    table = make_table(rng, lens, ps, 20, 10)
    for page in range(20):
        for t in range(ps):
            for which in range(2):
                x = rng.standard_normal((heads, d)) * 2.0 ** rng.integers(-spread, 1, (heads, d // 32)).repeat(32, axis=1)
                pool.put_values(which, page, np.arange(heads), t, x)
    q = encode(rng.standard_normal((2, heads * group, d)) * 2.0 ** rng.integers(-10, 3, (2, heads * group, d)), dtype)
    want, bound, _, _ = p4.ref_attention(q, pool, table, lens, 1.0, group, True)
    got, _ = _decode(gpu, pool, q, table, lens, scale=1.0)
    assert (np.abs(got - want) <= bound).all(), np.max(np.abs(got - want) / bound)


def test_scores_keep_f32s_accuracy(gpu):
    """One key's V is 1 and the others' 0, so O is a weight: its error is the score's, by which the three parts of Q can be told
    from two (2^-13 of the largest products) and the matrix product's fixed-point sums from coarser ones."""
    rng = np.random.default_rng(9)
    d, n = 128, 64
    pool = p4.Pool4(rng, 4, 1, 16, d, "f16")
    for page in range(4):
        for t in range(16):
            pool.put_values(1, page, 0, t, np.full(d, 1.0 if (page, t) == (1, 3) else 0.0))
    table = np.arange(4, dtype=np.int32)[None]
    q = _q(rng, 1, 16, d, "f16", 3.0)
    want, bound, _, _ = p4.ref_attention(q, pool, table, [n], 1 / np.sqrt(d), 16, True)
    got, _ = _decode(gpu, pool, q, table, [n])
    assert (np.abs(got - want) <= bound).all()
    # a product is off by 2 2^-24 of the sum of magnitudes, about 22 here, the scaled score by 2^-24 of itself, and a weight by its own
    # score's error and the others': 2 (2 * 22 + 10) 2^-24 = 6.5e-6
    assert np.max(np.abs(got - want) / want) < 1e-5


def test_equal_calls_give_equal_bits_and_the_workspace_serves_again(gpu):
    rng = np.random.default_rng(3)
    lens, heads, group, d, ps = [3000, 5, 0, 900], 2, 8, 64, 16
    pages = sum(-(-n // ps) for n in lens)
    pool = p4.Pool4(rng, pages, heads, ps, d)
    table = make_table(rng, lens, ps, pages, 188)
    q = _q(rng, 4, heads * group, d, "f16")
    o = nc.paged_options(num_seqs=4, num_q_heads=heads * group, max_pages=188, **pool.options())
    work = nc.DeviceBuffer(nc.paged4_workspace_bytes(o, mass=True))
    work.memset(0)
    mass = np.zeros((4, 188 * ps), np.float32)
    first = _decode(gpu, pool, q, table, lens, mass=mass, work=work)
    stream = nc.Stream()
    for _ in range(3):
        again = _decode(gpu, pool, q, table, lens, mass=mass, work=work, stream=stream.handle)
        assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])
