"""Paged cache on the GPU against references in float64 and in Python integers (pagedcheck.py, which also
derives the attention's error bound). Every place of the pools that no token fills holds NaN, and every table
entry past a request's length names no page, so reading either shows."""

import numpy as np
import pytest

import notcute_flash as nc
import pagedcheck as pc

pytestmark = pytest.mark.gpu


def say(msg):
    print(msg, flush=True)


def dev(x):
    return nc.DeviceBuffer.from_array(np.ascontiguousarray(x))


def fill(rng, pool, table, lens, sigma=1.0):
    """Random K and V rows for every token of every request."""
    for r, n in enumerate(lens):
        pos = np.arange(min(max(int(n), 0), table.shape[1] * pool.ps))
        page = table[r, pos // pool.ps] if len(pos) else np.zeros(0, dtype=np.int64)
        here = (page >= 0) & (page < pool.pages)
        for h in range(pool.heads):
            for which in (0, 1):
                x = rng.standard_normal((int(here.sum()), pool.d)) * (sigma if which == 0 else 1.0)
                pool.put(which, page[here], h, (pos % pool.ps)[here], pc.encode(x, pool.dtype))


def run_decode(gpu, pool, table, lens, q, opts, group, *, work=None, q_elem=0, o_elem=0, o_rows=None, stream=None):
    """Launches the attention and returns O of every place of its buffer, from o_elem on."""
    R, Hq, d = q.shape
    qs, os_ = opts.q_stride or Hq * d, opts.o_stride or Hq * d
    qbuf = np.full(q_elem + (R - 1) * qs + Hq * d, 0x7FFF, dtype=np.uint16)
    for r in range(R):
        qbuf[q_elem + r * qs:q_elem + r * qs + Hq * d] = q[r].ravel()
    rows = R if o_rows is None else o_rows
    o0 = np.full(o_elem + rows * os_, pc.SENTINEL, dtype=np.float32)
    own = work is None
    bufs = [dev(qbuf), dev(table), dev(np.asarray(lens, dtype=np.int32)), dev(o0)]
    k, v = pool.upload()
    work = nc.paged_workspace(opts) if own else work
    nc.paged_decode(gpu, pc.View(bufs[0], 2 * q_elem), k, v, bufs[1], bufs[2], pc.View(bufs[3], 4 * o_elem), work, opts,
                    stream)
    nc.synchronize()
    out = bufs[3].download(np.float32, o0.size)
    assert np.array_equal(out[:o_elem], o0[:o_elem])
    return out[o_elem:]


def check(out, ref, bound, opts, what):
    R, Hq, d = ref.shape
    os_ = opts.o_stride or Hq * d
    for r in range(R):
        got = out[r * os_:r * os_ + Hq * d].reshape(Hq, d)
        assert np.all(np.isfinite(got)), f"{what}: request {r} is not finite"
        over = np.abs(got - ref[r]) / bound[r]
        assert over.max() <= 1.0, f"{what}: request {r} off by {over.max():.2f} bounds at {np.unravel_index(over.argmax(), over.shape)}"
        assert np.all(out[r * os_ + Hq * d:(r + 1) * os_] == pc.SENTINEL), f"{what}: written behind request {r}"
    assert np.all(out[R * os_:] == pc.SENTINEL), f"{what}: rows behind the last request were written"


def decode_case(gpu, seed, lens, heads, group, d, ps, dtype="f16", layout="hnd", pad=0, sigma=1.0, scale=None, width=None,
                **kw):
    rng = np.random.default_rng(seed)
    held = [-(-max(n, 0) // ps) for n in lens]
    width = max(max(held), 1) if width is None else width
    pages = sum(min(h, width) for h in held) + 3
    pool = pc.Pool(rng, pages, heads, ps, d, dtype, layout, pad, poison=True)
    table = pc.make_table(rng, [min(max(n, 0), width * ps) for n in lens], ps, pages, width, spare=0x7FFFFFFF)
    fill(rng, pool, table, lens, sigma)
    q = pc.encode(rng.standard_normal((len(lens), heads * group, d)), dtype)
    strides = {k: kw.pop(k) for k in ("q_stride", "o_stride") if k in kw}
    opts = nc.paged_options(num_seqs=len(lens), num_q_heads=heads * group, max_pages=width, scale=scale, **strides,
                            **pool.options())
    say(f"[case] seed {seed} lens {lens[:6]} heads {heads}x{group} d {d} ps {ps} {dtype} {layout}")
    out = run_decode(gpu, pool, table, lens, q, opts, group, **kw)
    ref, bound = pc.ref_decode(q, pool, table, lens, opts.scale, group)
    check(out, ref, bound, opts, f"d {d} ps {ps} {dtype}")
    return out


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("ps", [16, 7])
def test_decode_lengths(gpu, d, ps, dtype):
    """One token to several tiles, the numbers around each tile's and page's end, and empty requests."""
    lens = [1, 0, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 0, 255, 256, 257, 511, 512, 513, 700]
    decode_case(gpu, 100 * d + ps, lens, 2, 2, d, ps, dtype)


@pytest.mark.parametrize("ps", [1, 2, 3, 8, 12, 24, 32, 48, 64, 100, 128, 1000])
def test_decode_page_sizes(gpu, ps):
    decode_case(gpu, ps, [333, 1, 0, 97, 250], 2, 4, 64, ps)
    decode_case(gpu, ps + 1, [130, 45], 3, 1, 32, ps, "bf16", layout="nhd")


@pytest.mark.parametrize("group", [1, 2, 3, 5, 7, 8, 15, 16, 17, 20, 32, 33, 48, 64, 65, 100, 130])
def test_decode_groups(gpu, group):
    decode_case(gpu, group, [200, 3, 0, 64], 2, group, 64, 16)
    decode_case(gpu, group + 500, [77], 1, group, 128, 24, "bf16")
    decode_case(gpu, group + 900, [150, 19], 3, group, 16, 16)


@pytest.mark.parametrize("layout", ["hnd", "nhd", "inter"])
@pytest.mark.parametrize("d", [16, 32, 64, 128])
def test_decode_layouts(gpu, layout, d):
    decode_case(gpu, d, [70, 300, 16], 3, 2, d, 16, layout=layout)
    decode_case(gpu, d + 1, [70, 300, 16], 3, 2, d, 10, "bf16", layout=layout)
    if layout != "inter":
        decode_case(gpu, d + 2, [70, 300, 16], 3, 2, d, 32, layout=layout, pad=8)


def test_decode_long(gpu):
    """Long requests: every workgroup has a share, and many join."""
    decode_case(gpu, 7, [40000], 1, 4, 64, 16)
    decode_case(gpu, 8, [20001, 5, 0, 9000], 2, 1, 128, 64, "bf16")
    decode_case(gpu, 9, [30011], 2, 8, 16, 16)
    decode_case(gpu, 10, [12345, 1, 20000], 2, 3, 32, 5)


@pytest.mark.parametrize("d,group,ps,dtype,pad", [(16, 1, 16, "f16", 0), (16, 3, 5, "bf16", 0), (32, 16, 16, "bf16", 1),
                                                  (32, 2, 7, "f16", 0), (64, 5, 16, "f16", 0), (64, 1, 24, "bf16", 3),
                                                  (128, 2, 32, "bf16", 0), (128, 16, 9, "f16", 0)])
def test_decode_many_short_heads(gpu, d, group, ps, dtype, pad):
    """More heads than workgroups, most of no more keys than a block: a workgroup's waves take one each, next to longer
    requests and empty ones. Lengths around a wave's step (32, 64) and a block (128, 256)."""
    lens = [1, 31, 32, 33, 0, 63, 64, 65, 100, 127, 128, 129, 2, 255, 256, 257, 17, 700, 0, 5, 16, 15, 90, 3, 48, 1]
    decode_case(gpu, 140 + d + group, lens, 43, group, d, ps, dtype, o_stride=43 * group * d + pad,
                q_stride=43 * group * d + 8 * pad)


@pytest.mark.parametrize("count", [63, 64, 65, 200, 257, 700, 1500])
def test_decode_many_requests(gpu, count):
    rng = np.random.default_rng(count)
    lens = np.exp(rng.uniform(0, np.log(300), count)).astype(int)
    lens[rng.random(count) < 0.2] = 0
    lens[-1] = 0
    decode_case(gpu, count, lens.tolist(), 1, 2, 32, 16)


def test_decode_more_requests_than_lanes_twice(gpu):
    """Over 64 requests a lane of the wave that finds a workgroup's first."""
    rng = np.random.default_rng(5)
    lens = rng.integers(0, 3, 4500)
    lens[[700, 4499]] = [900, 40]
    decode_case(gpu, 6, lens.tolist(), 1, 1, 16, 16)


def test_decode_wide_groups_over_long_requests(gpu):
    """Several waves on the same keys, heads in parts, and pieces to join."""
    decode_case(gpu, 14, [5000, 130], 1, 40, 64, 16)
    decode_case(gpu, 15, [3000, 0, 700], 2, 70, 128, 32, "bf16")
    decode_case(gpu, 16, [4001], 1, 64, 32, 5)
    decode_case(gpu, 17, [9000], 1, 20, 16, 16, "bf16")


@pytest.mark.parametrize("d,group,ps,dtype", [(16, 1, 16, "f16"), (16, 16, 3, "bf16"), (32, 4, 16, "f16"), (64, 8, 64, "bf16"),
                                              (64, 1, 100, "f16"), (128, 16, 16, "f16"), (128, 64, 16, "bf16"), (128, 33, 10, "f16")])
def test_decode_one_long_head(gpu, d, group, ps, dtype):
    """Every workgroup has a piece of the same few heads: pieces are added up in rounds."""
    for lens in ([70000], [33000, 1, 20000]):
        out = decode_case(gpu, d + group, lens, 1, group, d, ps, dtype)
        again = decode_case(gpu, d + group, lens, 1, group, d, ps, dtype)
        assert np.array_equal(out.view(np.uint32), again.view(np.uint32))


@pytest.mark.parametrize("d,group,ps", [(128, 1, 16), (64, 4, 16), (64, 2, 24), (32, 3, 7), (16, 8, 16)])
def test_decode_piece_counts(gpu, d, group, ps):
    """Lengths of 15 to 66 blocks of one head, a piece each: at the edges of what is added up at once."""
    block = 256 if d <= 32 else 128
    for blocks in (15, 16, 17, 31, 32, 33, 34, 63, 64, 65, 66):
        decode_case(gpu, blocks + d, [blocks * block - blocks % 3], 1, group, d, ps)


@pytest.mark.parametrize("d,heads,group,ps,layout,dtype", [
    (16, 4, 4, 16, "nhd", "f16"), (16, 2, 8, 1, "hnd", "bf16"), (16, 8, 3, 5, "nhd", "f16"), (16, 12, 1, 32, "inter", "bf16"),
    (32, 4, 2, 16, "nhd", "bf16"), (32, 6, 4, 7, "nhd", "f16"), (32, 4, 1, 1, "hnd", "f16"), (32, 2, 3, 16, "nhd", "f16"),
    (64, 4, 4, 16, "nhd", "f16"), (64, 8, 1, 1, "hnd", "bf16"), (64, 4, 3, 24, "nhd", "bf16"), (64, 12, 2, 64, "inter", "f16"),
    (128, 4, 4, 32, "nhd", "bf16"), (128, 8, 1, 10, "nhd", "f16"), (128, 4, 2, 1, "nhd", "bf16"), (128, 4, 3, 16, "inter", "f16")])
def test_decode_heads_beside_each_other(gpu, d, heads, group, ps, layout, dtype):
    """Token-major pages, where waves take neighbouring heads: ragged requests with empty ones, a long one whose pieces
    are added up, strides and alignments, an absent page in the middle."""
    lens = [1, 0, 31, 33, 64, 65, 129, 700, 2000, 5, 257, 32, 63, 0]
    seed = 700 + d + heads + group + ps
    decode_case(gpu, seed, lens, heads, group, d, ps, dtype, layout, width=3000 // ps)
    decode_case(gpu, seed + 1, lens, heads, group, d, ps, dtype, layout, width=3000 // ps, pad=8, sigma=4.0,
                q_stride=heads * group * d + 3, o_stride=heads * group * d + 1, q_elem=1, o_elem=3)
    first, again = (decode_case(gpu, seed + 2, [20011, 3], heads, group, d, ps, dtype, layout) for _ in range(2))
    assert np.array_equal(first.view(np.uint32), again.view(np.uint32))
    rng = np.random.default_rng(seed)
    n, width = 900, -(-1000 // ps)
    held = -(-n // ps)
    pool = pc.Pool(rng, held + 2, heads, ps, d, dtype, layout)
    table = pc.make_table(rng, [n], ps, held + 2, width, spare=-1)
    table[0, held // 2] = held + 2  # names no page
    q = pc.encode(rng.standard_normal((1, heads * group, d)), dtype)
    opts = nc.paged_options(num_seqs=1, num_q_heads=heads * group, max_pages=width, **pool.options())
    out = run_decode(gpu, pool, table, [n], q, opts, group)
    ref, bound = pc.ref_decode(q, pool, table, [n], opts.scale, group)
    check(out, ref, bound, opts, "absent page")


def test_decode_leaves_the_counters_at_zero(gpu):
    opts = nc.paged_options(num_seqs=2, num_q_heads=4, num_kv_heads=2, head_dim=64, page_size=16, num_pages=2000, max_pages=1000)
    work = nc.paged_workspace(opts)
    for seed, lens in ((1, [15000, 300]), (2, [40, 16000]), (3, [0, 5])):
        decode_case(gpu, seed, lens, 2, 2, 64, 16, work=work)
        assert not np.any(work.download(np.uint32, 10240)), "a counter of the workspace is not 0"


def test_decode_and_build_table_strides(gpu):
    """Rows of the table apart from each other: what stands between them is neither read nor written."""
    rng = np.random.default_rng(18)
    lens, ps, width, stride = [50, 0, 33], 16, 4, 11
    pool = pc.Pool(rng, 12, 2, ps, 64)
    table = pc.make_table(rng, lens, ps, 12, width)
    wide = np.full((3, stride), 0x7FFFFFF0, dtype=np.int32)
    wide[:, :width] = table
    q = pc.encode(rng.standard_normal((3, 4, 64)), "f16")
    opts = nc.paged_options(num_seqs=3, num_q_heads=4, max_pages=width, table_stride=stride, **pool.options())
    flat = wide.ravel()[:2 * stride + width]  # no longer than has to be
    out = run_decode(gpu, pool, flat, lens, q, opts, 2)
    ref, bound = pc.ref_decode(q, pool, table, lens, opts.scale, 2)
    check(out, ref, bound, opts, "table stride")
    tab, free = dev(flat), np.arange(12, dtype=np.int32)
    bopts = nc.paged_options(num_seqs=3, head_dim=64, page_size=ps, num_pages=12, max_pages=width, table_stride=stride)
    cached, new = np.array(lens), np.array([10, 20, 31])
    outs = [nc.DeviceBuffer(4 * n) for n in (3, 4, 61, 4)]
    nc.paged_build(gpu, dev(cached.astype(np.int32)), dev(new.astype(np.int32)), dev(free), dev(np.zeros(1, np.int32)), tab, *outs, bopts)
    nc.synchronize()
    want = pc.ref_build(cached, new, free, 0, table, 61, ps, 12)
    wide[:, :width] = want[0]
    assert np.array_equal(tab.download(np.int32, flat.size), wide.ravel()[:flat.size])
    assert np.array_equal(outs[2].download(np.int32, 61), want[3])


def test_decode_all_empty(gpu):
    out = decode_case(gpu, 3, [0, 0, 0], 2, 2, 64, 16)
    assert np.all(out == 0.0)
    out = decode_case(gpu, 3, [-5, 0], 2, 20, 64, 16)
    assert np.all(out == 0.0)


def test_decode_strides_and_alignment(gpu):
    for q_elem, o_elem in ((1, 1), (3, 2), (8, 3)):
        decode_case(gpu, 20 + q_elem, [90, 0, 33], 2, 3, 64, 16, q_elem=q_elem, o_elem=o_elem, q_stride=6 * 64 + 5,
                    o_stride=6 * 64 + 7)
    decode_case(gpu, 31, [90, 5], 2, 3, 16, 16, "bf16", q_elem=5, o_elem=1)
    decode_case(gpu, 32, [90, 5], 1, 1, 128, 16, o_rows=9)


@pytest.mark.parametrize("sigma,scale", [(1.0, 0.0), (1.0, -0.5), (6.0, None), (30.0, 1.0), (0.01, None)])
def test_decode_scales_and_peaks(gpu, sigma, scale):
    """Flat, reversed and peaked weights (sigma 30: one key has all of it)."""
    for dtype in ("f16", "bf16"):
        decode_case(gpu, 41, [600, 47, 1], 2, 2, 64, 16, dtype, sigma=sigma, scale=scale)


def test_decode_lengths_past_the_table(gpu):
    """A length is cut to what the table's row can hold; one that is negative counts as 0."""
    decode_case(gpu, 51, [100, 2 ** 31 - 1, -1, -2 ** 31, 49], 2, 2, 64, 16, width=3)


def test_decode_bad_pages(gpu):
    """Entries outside the pool are absent keys: here and there, all of a request's, the last of a page run."""
    for ps in (16, 5, 64):
        rng = np.random.default_rng(60 + ps)
        lens = [200, 90, 64, 130]
        held = [-(-n // ps) for n in lens]
        pages = sum(held)
        pool = pc.Pool(rng, pages, 2, ps, 64, poison=True)
        table = pc.make_table(rng, lens, ps, pages, max(held))
        table[0, ::3] = [-1, pages, 2 ** 31 - 1, -2 ** 31, -7][ps % 5]
        table[1, :] = pages
        table[2, held[2] - 1] = -1
        table[3, 0] = -2 ** 31
        fill(rng, pool, table, lens)
        q = pc.encode(rng.standard_normal((4, 6, 64)), "f16")
        opts = nc.paged_options(num_seqs=4, num_q_heads=6, max_pages=max(held), **pool.options())
        out = run_decode(gpu, pool, table, lens, q, opts, 3)
        ref, bound = pc.ref_decode(q, pool, table, lens, opts.scale, 3)
        check(out, ref, bound, opts, f"bad pages, ps {ps}")
        assert np.all(out[6 * 64:2 * 6 * 64] == 0.0)


def test_decode_infinite_scores(gpu):
    """K of -infinity takes a key out (its weight is exactly 0); where every key is out, O is 0. A NaN among the
    keys that count is not hidden."""
    for dtype, d in (("f16", 64), ("bf16", 128), ("f16", 16)):
        rng = np.random.default_rng(70 + d)
        pool = pc.Pool(rng, 12, 1, 16, d, dtype)
        table = np.arange(12, dtype=np.int32).reshape(3, 4)
        lens = [60, 64, 40]
        q = np.abs(rng.standard_normal((3, 2, d))) + 0.1
        inf = pc.encode(np.full((1, d), -np.inf), dtype)
        keep = {0: np.array([3, 17, 40, 59]), 1: np.array([], dtype=int), 2: np.arange(40)}
        for r in range(3):
            for j in range(lens[r]):
                if j not in keep[r]:
                    pool.put(0, table[r, j // 16], 0, j % 16, inf[0])
        pool.put(0, table[2, 1], 0, 5, pc.encode(np.full(d, np.nan), dtype))
        qb = pc.encode(q, dtype)
        opts = nc.paged_options(num_seqs=3, num_q_heads=2, max_pages=4, **pool.options())
        out = run_decode(gpu, pool, table, lens, qb, opts, 2).reshape(3, 2, d)
        assert np.all(out[1] == 0.0)
        assert np.all(np.isnan(out[2]))
        kept = pc.Pool(rng, 1, 1, 4, d, dtype)
        for i, j in enumerate(keep[0]):
            for which in (0, 1):
                kept.put(which, 0, 0, i, pool.get(which, table[0, j // 16], 0, j % 16))
        ref, bound = pc.ref_decode(qb[:1], kept, np.array([[0]], dtype=np.int32), [4], opts.scale, 2)
        assert np.all(np.abs(out[0] - ref[0]) <= bound[0])


@pytest.mark.parametrize("d,dtype", [(16, "bf16"), (128, "bf16"), (64, "f16")])
def test_decode_sums_at_the_largest_value(gpu, d, dtype):
    """200000 keys of one score and V at the type's largest value: O is that value, and no sum on the way passes
    f32's range. The weights are one power of two, so their sums are exact; O is added up in at most 200000/32
    steps of a wave, 4 waves and 1024 pieces, 2^-24 each, and the quotient is within 2^-22."""
    n, pages = 200000, 4
    rng = np.random.default_rng(72)
    pool = pc.Pool(rng, pages, 1, 16, d, dtype)
    most = 3.3895313892515355e38 if dtype == "bf16" else 65504.0
    for p in range(pages):
        for t in range(16):
            pool.put(1, p, 0, t, pc.encode(np.full(d, most), dtype))
    table = (np.arange(n // 16, dtype=np.int32) % pages).reshape(1, -1)
    q = np.zeros((1, 2, d), dtype=np.uint16)
    opts = nc.paged_options(num_seqs=1, num_q_heads=2, max_pages=n // 16, **pool.options())
    out = run_decode(gpu, pool, table, [n], q, opts, 2).astype(np.float64)
    assert np.all(np.abs(out / most - 1.0) <= (n / 32 + 4 + 1024) * 2.0 ** -24 + 2.0 ** -22)


def test_decode_shared_pages(gpu):
    """Two requests with a common prefix read the same pages."""
    rng = np.random.default_rng(80)
    pool = pc.Pool(rng, 9, 2, 16, 64)
    table = np.array([[4, 2, 7, 0], [4, 2, 8, 1], [4, 2, 7, 0]], dtype=np.int32)
    lens = [60, 64, 60]
    q = pc.encode(rng.standard_normal((1, 4, 64)).repeat(3, axis=0), "f16")
    opts = nc.paged_options(num_seqs=3, num_q_heads=4, max_pages=4, **pool.options())
    out = run_decode(gpu, pool, table, lens, q, opts, 2)
    ref, bound = pc.ref_decode(q, pool, table, lens, opts.scale, 2)
    check(out, ref, bound, opts, "shared pages")


def test_decode_repeats_and_shares_a_workspace(gpu):
    """Equal calls give equal bits, and one workspace serves calls of other options in between."""
    big = dict(seed=90, lens=[9000, 100], heads=2, group=4, d=64, ps=16)
    small = dict(seed=91, lens=[700, 3000, 12], heads=1, group=1, d=128, ps=24, dtype="bf16")
    # large enough for both
    work = nc.DeviceBuffer(max(nc.paged_workspace_bytes(nc.paged_options(
        num_seqs=3, num_q_heads=g * h, num_kv_heads=h, head_dim=d, page_size=16, num_pages=1000, max_pages=600))
        for g, h, d in ((4, 2, 64), (1, 1, 128))))
    work.memset(0)
    first = [decode_case(gpu, work=work, **c) for c in (big, small)]
    for _ in range(3):
        for c, f in zip((small, big), first[::-1]):
            assert np.array_equal(decode_case(gpu, work=work, **c).view(np.uint32), f.view(np.uint32))


def test_decode_offsets_past_32_bits(gpu):
    """Pages 4 GiB apart: element offsets past 2^32, byte offsets past 2^33."""
    rng = np.random.default_rng(99)
    ps, d, heads = 16, 64, 2
    stride = 2 ** 31 + 64
    small = pc.Pool(rng, 3, heads, ps, d)  # the same pages, close together
    opts = nc.paged_options(num_seqs=2, num_q_heads=4, num_kv_heads=heads, head_dim=d, page_size=ps, num_pages=3,
                            max_pages=2, page_stride=stride)
    span = heads * ps * d
    caches = [nc.DeviceBuffer(2 * (2 * stride + span)) for _ in range(2)]
    table = np.array([[2, 0], [1, 2]], dtype=np.int32)
    lens = [25, 32]
    q = pc.encode(rng.standard_normal((2, 4, d)), "f16")
    for which in (0, 1):
        for p in range(3):
            caches[which].upload(small.bufs[which][p * span:(p + 1) * span], 2 * p * stride)
    bufs = [dev(q), dev(table), dev(np.array(lens, np.int32)), nc.DeviceBuffer(2 * 4 * d * 4)]
    work = nc.paged_workspace(opts)
    nc.paged_decode(gpu, bufs[0], *caches, bufs[1], bufs[2], bufs[3], work, opts)
    nc.synchronize()
    ref, bound = pc.ref_decode(q, small, table, lens, opts.scale, 2)
    check(bufs[3].download(np.float32, 2 * 4 * d), ref, bound, opts, "far pages")
    # a row into the last page, next to the end of the cache
    rows = [pc.encode(rng.standard_normal((1, heads, d)), "f16") for _ in range(2)]
    slots = dev(np.array([2 * ps + ps - 1], np.int32))
    nc.paged_append(gpu, dev(rows[0]), dev(rows[1]), slots, *caches, opts)
    nc.synchronize()
    for which in (0, 1):
        got = caches[which].download(np.uint16, span, 2 * 2 * stride)
        want = small.bufs[which][2 * span:3 * span].copy().reshape(heads, ps, d)
        want[:, ps - 1] = rows[which][0]
        assert np.array_equal(got, want.ravel())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("layout", ["hnd", "nhd", "inter"])
@pytest.mark.parametrize("ps,heads,shift,extra", [(16, 2, 0, 0), (7, 3, 1, 3), (1, 1, 0, 8), (24, 5, 2, 2), (32, 8, 4, 0)])
def test_append(gpu, layout, d, dtype, ps, heads, shift, extra):
    """Rows at any alignment and stride into every layout, padding skipped, everything else left alone."""
    rng = np.random.default_rng(d + ps)
    pages, n = 11, 9 * ps - 3 if ps > 1 else 9
    pool = pc.Pool(rng, pages, heads, ps, d, dtype, layout, 8 if layout == "nhd" else 0)
    slots = rng.permutation(pages * ps)[:n].astype(np.int32)
    slots[rng.random(n) < 0.2] = -1
    slots[n // 2] = pages * ps       # not in the pool either
    slots[n // 3] = -2 ** 31
    stride = heads * d + extra
    src = [rng.integers(0, 2 ** 16, shift + n * stride + 3).astype(np.uint16) for _ in range(2)]
    opts = nc.paged_options(row_stride=stride, num_q_heads=heads, **pool.options())
    k, v = pool.upload()
    bufs = [dev(src[0]), dev(src[1]), dev(slots)]
    nc.paged_append(gpu, pc.View(bufs[0], 2 * shift), pc.View(bufs[1], 2 * shift), bufs[2], k, v, opts)
    nc.synchronize()
    for i, slot in enumerate(slots):
        if 0 <= slot < pages * ps:
            for which in (0, 1):
                row = src[which][shift + i * stride:shift + i * stride + heads * d].reshape(heads, d)
                pool.put(which, slot // ps, np.arange(heads), slot % ps, row)
    for got, want in zip(pool.download(k, v), pool.bufs):
        assert np.array_equal(got, want)


def test_append_of_fewer_rows_and_head_strides(gpu):
    """The first rows only; heads of a row apart from each other, from one [k, v]-interleaved buffer."""
    rng = np.random.default_rng(5)
    pool = pc.Pool(rng, 4, 3, 16, 32)
    src = rng.integers(0, 2 ** 16, 40 * 3 * 64).astype(np.uint16)  # [row][head][k, v][32]
    slots = rng.permutation(64)[:40].astype(np.int32)
    opts = nc.paged_options(num_q_heads=3, row_head_stride=64, **pool.options())
    k, v = pool.upload()
    buf = dev(src)
    nc.paged_append(gpu, buf, pc.View(buf, 64), dev(slots), k, v, opts, num_rows=33)
    nc.synchronize()
    rows = src.reshape(40, 3, 2, 32)
    for i in range(33):
        for which in (0, 1):
            pool.put(which, slots[i] // 16, np.arange(3), slots[i] % 16, rows[i, :, which])
    for got, want in zip(pool.download(k, v), pool.bufs):
        assert np.array_equal(got, want)


def run_build(gpu, cached, new, free, cursor, table, places, ps, num_pages, in_place=False, stream=None):
    R, width = table.shape
    opts = nc.paged_options(num_seqs=R, head_dim=64, page_size=ps, num_pages=num_pages, max_pages=width)
    lens = dev(cached.astype(np.int32))
    counts = dev(np.array([cursor, 77, 77, 77, 77], np.int32))
    cur = pc.View(counts, 0, 4) if in_place else dev(np.array([cursor], np.int32))
    out_lens = lens if in_place else dev(np.full(R, 77, np.int32))
    tab, off, slots = dev(table), dev(np.full(R + 3, 77, np.int32)), dev(np.full(places + 5, 77, np.int32))
    nc.paged_build(gpu, lens, dev(new.astype(np.int32)), dev(free.astype(np.int32)), cur, tab, out_lens,
                   off, pc.View(slots, 0, 4 * places), counts, opts, stream)
    nc.synchronize()
    got = (tab.download(np.int32, table.size).reshape(table.shape), out_lens.download(np.int32, R),
           off.download(np.int32, R + 3), slots.download(np.int32, places + 5), counts.download(np.int32, 5))
    assert np.all(got[2][R + 1:] == 77) and np.all(got[3][places:] == 77) and got[4][4] == 77
    return got[0], got[1], got[2][:R + 1], got[3][:places], got[4][:4]


def build_case(gpu, seed, R, ps, width, max_cached, max_new, places=None, spare=10, cursor=0, in_place=False, wild=False):
    rng = np.random.default_rng(seed)
    cap = width * ps
    cached = rng.integers(0, max_cached + 1, R).clip(max=cap)
    new = rng.integers(0, max_new + 1, R)
    if wild:  # some that cannot be
        cached[rng.random(R) < 0.05] = -3
        cached[rng.random(R) < 0.05] = 2 ** 31 - 1
        new[rng.random(R) < 0.05] = -2 ** 31
        new[rng.random(R) < 0.05] = 2 ** 31 - 1
    held = np.minimum(-(-np.maximum(cached, 0) // ps), width)
    need = np.minimum(-(-(np.maximum(cached, 0) + np.maximum(new, 0)) // ps), width)
    pages = int(need.sum()) + 20
    ids = rng.permutation(pages)
    table = np.full((R, width), -1, dtype=np.int32)
    at = 0
    for r, h in enumerate(held):
        table[r, :h] = ids[at:at + h]
        at += h
    free = np.concatenate([rng.integers(0, pages, cursor), ids[at:]])
    free = free[:max(0, cursor + int((need - held).sum()) + spare)]
    total = int(np.maximum(new, 0).sum())
    places = total + 7 if places is None else places
    say(f"[case] build R {R} ps {ps} width {width} rows {total} places {places} free {len(free)} in place {in_place}")
    got = run_build(gpu, cached, new, free, cursor, table, places, ps, pages, in_place)
    want = pc.ref_build(cached, new, free, cursor, table, places, ps, pages)
    for name, g, w in zip(("table", "lens", "offsets", "slots", "counts"), got, want):
        assert np.array_equal(g, w), f"{name}: differs at {np.argwhere(np.asarray(g) != np.asarray(w))[:5].ravel()}"
    return want


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("R,ps,width,max_new,places", [
    (1, 16, 300, 4000, None), (1, 1, 70, 64, 64), (1, 1, 70, 64, 65), (3, 32, 129, 946, 1600), (8, 7, 80, 100, 4096),
    (60, 16, 30, 200, 128), (64, 24, 9, 8, 512), (64, 24, 9, 9, 513), (65, 16, 9, 9, 521), (2, 16, 9, 1, 5000)])
def test_build_few_requests_many_slots(gpu, R, ps, width, max_new, places, in_place):
    """Where a step's slots go from one workgroup to several, and slot maps with much padding or too few places."""
    build_case(gpu, 500 + R + ps, R, ps, width, 50, max_new, places=places, cursor=4, in_place=in_place)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("R,ps,width,max_cached,max_new", [
    (1, 16, 4, 0, 1), (1, 16, 4, 40, 0), (5, 1, 40, 20, 3), (64, 16, 64, 900, 1), (255, 7, 30, 100, 9),
    (256, 16, 8, 100, 1), (257, 64, 3, 150, 2), (1000, 16, 20, 200, 5), (1024, 24, 9, 99, 1), (1025, 16, 9, 99, 2),
    (3000, 16, 5, 40, 3), (40, 16, 300, 1000, 3000), (300, 128, 40, 2000, 700), (2500, 16, 30, 100, 60)])
def test_build(gpu, R, ps, width, max_cached, max_new, in_place):
    build_case(gpu, R + ps, R, ps, width, max_cached, max_new, in_place=in_place)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("R,max_new", [(50, 40), (700, 90), (2000, 30)])
def test_build_refuses_requests(gpu, R, max_new, in_place):
    """The list runs out, the slot map is too short, the table too narrow, lengths that cannot be."""
    assert build_case(gpu, 1, R, 16, 10, 100, max_new, spare=-R // 3, in_place=in_place)[4][3] > 0
    assert build_case(gpu, 2, R, 16, 10, 100, max_new, places=R * max_new // 4, in_place=in_place)[4][3] > 0
    assert build_case(gpu, 3, R, 16, 7, 112, max_new, in_place=in_place)[4][3] > 0
    assert build_case(gpu, 4, R, 5, 20, 60, max_new, wild=True, places=R * max_new, in_place=in_place)[4][3] > 0
    build_case(gpu, 5, R, 16, 12, 100, max_new, cursor=9, in_place=in_place)
    build_case(gpu, 6, R, 16, 12, 100, max_new, places=0, in_place=in_place)


def test_build_no_list_and_bad_ids(gpu):
    one = np.array([[3, -1]], dtype=np.int32)
    got = run_build(gpu, np.array([4]), np.array([4]), np.array([], np.int32), 0, one, 6, 16, 5)
    assert got[1][0] == 8 and got[3].tolist() == [52, 53, 54, 55, -1, -1] and got[4].tolist() == [0, 4, 0, 0]
    for bad in (-1, 5, 2 ** 31 - 1, -2 ** 31):  # a listed page that is not in the pool: entered, but no slots
        got = run_build(gpu, np.array([15]), np.array([3]), np.array([bad]), 0, one, 3, 16, 5)
        assert got[0].tolist() == [[3, bad]] and got[3].tolist() == [63, -1, -1] and got[4].tolist() == [1, 3, 1, 0]
    # a cursor that is negative counts as 0, one past the list leaves nothing
    got = run_build(gpu, np.array([16]), np.array([1]), np.array([4]), -3, one, 1, 16, 5)
    assert got[0].tolist() == [[3, 4]] and got[3].tolist() == [64] and got[4].tolist() == [1, 1, 1, 0]
    got = run_build(gpu, np.array([16]), np.array([1]), np.array([4]), 1, one, 1, 16, 5)
    assert got[0].tolist() == [[3, -1]] and got[3].tolist() == [-1] and got[4].tolist() == [1, 1, 0, 1]


class Serving:
    """A few layers' caches and a step of them: build, then append and decode per layer."""

    def __init__(self, seed, R=5, heads=2, group=3, d=64, ps=16, width=12, dtype="f16", layers=2, pages=40):
        self.rng = np.random.default_rng(seed)
        self.R, self.heads, self.group, self.d, self.ps, self.dtype = R, heads, group, d, ps, dtype
        self.opts = nc.paged_options(num_seqs=R, num_q_heads=heads * group, num_kv_heads=heads, head_dim=d, page_size=ps,
                                     num_pages=pages, max_pages=width, dtype=dtype)
        self.pools = [pc.Pool(self.rng, pages, heads, ps, d, dtype, poison=True) for _ in range(layers)]
        self.caches = [p.upload() for p in self.pools]
        self.free = dev(self.rng.permutation(pages).astype(np.int32))
        self.lens, self.counts = dev(np.zeros(R, np.int32)), dev(np.zeros(4, np.int32))
        self.table = dev(np.full((R, width), -1, np.int32))
        self.work = nc.paged_workspace(self.opts)
        self.length = np.zeros(R, dtype=int)
        self.history = [[[] for _ in range(R)] for _ in range(layers)]  # (k, v) rows of each request

    def prepare(self, new, places):
        """The step's inputs: lengths, rows of K, V and Q per layer."""
        self.new = np.asarray(new)
        rows = int(self.new.sum())
        self.places = places
        self.k = [pc.encode(self.rng.standard_normal((places, self.heads, self.d)), self.dtype) for _ in self.pools]
        self.v = [pc.encode(self.rng.standard_normal((places, self.heads, self.d)), self.dtype) for _ in self.pools]
        self.q = [pc.encode(self.rng.standard_normal((self.R, self.heads * self.group, self.d)), self.dtype) for _ in self.pools]
        at = np.concatenate([[0], np.cumsum(self.new)])
        for layer, h in enumerate(self.history):
            for r in range(self.R):
                h[r] += [(self.k[layer][i], self.v[layer][i]) for i in range(at[r], at[r + 1])]
        self.length += self.new
        return rows

    def upload(self):
        if not hasattr(self, "dnew"):
            self.dnew, self.off = nc.DeviceBuffer(4 * self.R), nc.DeviceBuffer(4 * self.R + 4)
            self.slots = nc.DeviceBuffer(4 * self.places)
            self.dk, self.dv, self.dq, self.do = ([nc.DeviceBuffer(n) for _ in self.pools] for n in (
                self.k[0].nbytes, self.k[0].nbytes, self.q[0].nbytes, 2 * self.q[0].nbytes))
        self.dnew.upload(self.new.astype(np.int32))
        for i in range(len(self.pools)):
            self.dk[i].upload(self.k[i])
            self.dv[i].upload(self.v[i])
            self.dq[i].upload(self.q[i])
            self.do[i].memset(0xFF)

    def launch(self, gpu, stream=None):
        nc.paged_build(gpu, self.lens, self.dnew, self.free, pc.View(self.counts, 0, 4), self.table, self.lens, self.off,
                       self.slots, self.counts, self.opts, stream)
        for i, (k, v) in enumerate(self.caches):
            nc.paged_append(gpu, self.dk[i], self.dv[i], self.slots, k, v, self.opts, stream)
            nc.paged_decode(gpu, self.dq[i], k, v, self.table, self.lens, self.do[i], self.work, self.opts, stream)

    def verify(self, what):
        assert np.array_equal(self.lens.download(np.int32, self.R), self.length), what
        for i in range(len(self.pools)):
            out = self.do[i].download(np.float32, self.q[i].size).reshape(self.q[i].shape)
            for r in range(self.R):
                n = int(self.length[r])
                flat = pc.Pool(self.rng, 1, self.heads, max(n, 1), self.d, self.dtype)
                for j, (k, v) in enumerate(self.history[i][r]):
                    flat.put(0, 0, np.arange(self.heads), j, k)
                    flat.put(1, 0, np.arange(self.heads), j, v)
                ref, bound = pc.ref_decode(self.q[i][r:r + 1], flat, np.zeros((1, 1), np.int32), [n], self.opts.scale, self.group)
                assert np.all(np.abs(out[r] - ref[0]) <= bound[0]), f"{what}: layer {i} request {r}"


@pytest.mark.parametrize("dtype,d,ps", [("f16", 64, 16), ("bf16", 128, 7), ("f16", 32, 24)])
def test_steps_together(gpu, dtype, d, ps):
    """Prompts, then single tokens (some requests idle), eagerly: tables, caches and attention follow."""
    s = Serving(7 + d, d=d, ps=ps, dtype=dtype, width=-(-190 // ps), pages=-(-800 // ps))
    s.prepare([50, 0, 17, 1, 90], 160)
    s.upload()
    s.launch(gpu)
    nc.synchronize()
    s.verify("prompts")
    for step in range(6):
        s.prepare([1, step % 2, 1, 0, 1] if step < 5 else [30, 2, 0, 1, 0], 160)
        s.upload()
        s.launch(gpu)
        nc.synchronize()
        s.verify(f"step {step}")


def test_captured_step_replays(gpu):
    """One captured step, replayed: lengths, tables, cursor and caches advance in place, with eager work of another
    shape and synchronisations between the replays, each of which is checked."""
    s = Serving(11, layers=3)
    s.prepare([20, 3, 0, 33, 15], 80)
    s.upload()
    s.launch(gpu)
    nc.synchronize()
    s.verify("prompts")
    stream = nc.Stream()
    graph = nc.Graph.capture(stream, lambda: s.launch(gpu, stream.handle))
    try:
        for step in range(20):
            s.prepare([1, 1, int(step > 3), 1, int(step % 3 == 0)], 80)
            s.upload()
            decode_case(gpu, 1000 + step, [300, 5], 1, 2, 32, 16)  # eager work between the replays
            graph.launch(stream)
            stream.synchronize()
            s.verify(f"replay {step}")
    finally:
        graph.destroy()
        stream.destroy()


def test_first_launches_captured(gpu):
    """A fresh module whose first launch of each kernel is recorded into a graph, which is then replayed with eager work in
    between."""
    module = nc.Module.load_embedded()
    s = Serving(13, d=32, ps=16, dtype="bf16", heads=4, width=40, pages=60)
    s.prepare([30, 0, 100, 7, 1], 150)
    s.upload()
    stream = nc.Stream()
    graph = nc.Graph.capture(stream, lambda: s.launch(module, stream.handle))
    try:
        for step, new in enumerate(([30, 0, 100, 7, 1], [1, 1, 1, 0, 1], [3, 1, 0, 1, 1], [1, 1, 1, 1, 1])):
            if step:
                s.prepare(new, 150)
                s.upload()
            decode_case(gpu, 1100 + step, [500, 70], 2, 2, 32, 7)
            graph.launch(stream)
            stream.synchronize()
            s.verify(f"replay {step}")
    finally:
        graph.destroy()
        stream.destroy()
        module.unload()


def test_two_threads_launch_through_one_module(gpu):
    """Two host threads at once, each with a stream, buffers and a workspace of its own."""
    import threading

    module = nc.Module.load_embedded()
    sides = [Serving(21 + i, d=64 if i else 128, ps=16, layers=1, width=30, pages=80) for i in range(2)]
    streams = [nc.Stream() for _ in sides]
    errors = []

    def steps(s, stream):
        try:
            for new in ([40, 0, 300, 7, 1], [1, 1, 1, 0, 1], [1, 1, 1, 1, 1], [2, 0, 1, 1, 9]):
                s.prepare(new, 360)
                s.upload()
                s.launch(module, stream.handle)
                stream.synchronize()
                s.verify("thread")
        except BaseException as e:  # shown by the main thread
            errors.append(e)

    threads = [threading.Thread(target=steps, args=x) for x in zip(sides, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for stream in streams:
        stream.destroy()
    module.unload()
    assert not errors, errors


def test_two_streams_with_workspaces_of_their_own(gpu):
    """Calls that overlap in time, each with its own workspace, give what they give alone."""
    rng = np.random.default_rng(12)
    sides = []
    for i in range(2):
        ps, d, lens = 16, 64, [6000 + 100 * i, 900]
        held = [-(-n // ps) for n in lens]
        pool = pc.Pool(rng, sum(held), 2, ps, d)
        table = pc.make_table(rng, lens, ps, sum(held), max(held))
        q = pc.encode(rng.standard_normal((2, 8, d)), "f16")
        opts = nc.paged_options(num_seqs=2, num_q_heads=8, max_pages=max(held), **pool.options())
        sides.append((opts, dev(q), *pool.upload(), dev(table), dev(np.array(lens, np.int32)),
                      nc.DeviceBuffer(q.size * 4), nc.paged_workspace(opts), nc.Stream(), pool, table, lens, q))
    for _ in range(20):
        for opts, q, k, v, t, n, o, w, st, *_ in sides:
            nc.paged_decode(gpu, q, k, v, t, n, o, w, opts, st.handle)
    for opts, q, k, v, t, n, o, w, st, pool, table, lens, qh in sides:
        st.synchronize()
        ref, bound = pc.ref_decode(qh, pool, table, lens, opts.scale, 4)
        check(o.download(np.float32, qh.size), ref, bound, opts, "two streams")
        st.destroy()


def test_decode_continues_a_flash_prompt(gpu):
    """The prompt by the flash forward, its K and V into the cache, then the last token again by decode: the same
    row of the same attention, within the two paths' bars."""
    import flashcheck as fc

    S, heads, d = 77, 4, 64
    rng = np.random.default_rng(13)
    q, k, v = (pc.encode(rng.standard_normal((heads, S, d)), "f16") for _ in range(3))
    fo = nc.options(seq_len=S, head_dim=d, batch_heads=heads, causal=True)
    dq, dk, dv, do = dev(q), dev(k), dev(v), nc.DeviceBuffer(heads * S * d * 4)
    nc.flash_launch(gpu, dq, dk, dv, do, fo)
    pages = -(-S // 16)
    # K and V of the prompt are [head][token][dim]: a row's heads stand S*d apart
    opts = nc.paged_options(num_q_heads=heads, head_dim=d, page_size=16, num_pages=pages, max_pages=pages, row_stride=d,
                            row_head_stride=S * d, q_head_stride=S * d, q_stride=heads * S * d)
    kc, vc = (nc.DeviceBuffer(pages * heads * 16 * d * 2) for _ in range(2))
    order = rng.permutation(pages).astype(np.int32)
    slots = dev((order[np.arange(S) // 16] * 16 + np.arange(S) % 16).astype(np.int32))
    nc.paged_append(gpu, dk, dv, slots, kc, vc, opts)
    out = nc.DeviceBuffer(heads * d * 4)
    nc.paged_decode(gpu, pc.View(dq, 2 * (S - 1) * d), kc, vc, dev(order[None]), dev(np.array([S], np.int32)), out,
                    nc.paged_workspace(opts), opts)
    nc.synchronize()
    last = do.download(np.float32, heads * S * d).reshape(heads, S, d)[:, -1]
    assert np.max(np.abs(out.download(np.float32, heads * d).reshape(heads, d) - last)) <= fc.MAX_ABS


def test_harness_command(gpu, capsys):
    """flash_harness.py paged: prompts and decoding steps over a paged cache, a record per case, each within its
    tolerance."""
    import json

    import flash_harness as fh

    assert fh.main(["paged", "--warmup", "1", "--iters", "3"]) == 0
    recs = [json.loads(line) for line in capsys.readouterr().out.splitlines() if line.startswith("{")]
    assert len(recs) == len(fh.PAGED_CASES)
    for r in recs:
        assert set(r) == set(fh.RECORD_KEYS) and r["kernel"] == "paged_attention"
        assert r["correct"] and r["max_abs_error"] <= fh.PAGED_TOL and r["min_ms"] > 0
