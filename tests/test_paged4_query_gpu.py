"""Queries of a 4-bit cache's attention whose values are far apart: a few large channels among ordinary ones, and very small values. The
weights themselves are compared (as masses, one query head each), and O, with float64.

Bound of a score, in the exponent's natural units: an instruction's sum of 128 exact products has at most 8 roundings of 2^-24 of
their magnitudes (test_hw_fp4_gpu.py), and the products of up to 4 parts of Q are added up in f32: 16 2^-24 sum |q_i k_i| covers them. The scale, its
product and the difference to the maximum are 2 2^-23 of the score's own size and 2^-24 of the difference. What the parts leave of q_i is at
most 2^-25 of the largest of its 32 values. A weight p_j has its own score's error and at most as much by the others',
2 2^-22 by exponentials (its own and those of the sum), and what the running maxima cost: 2^-22 for each of at most 12."""

import numpy as np
import pytest

import notcute_flash as nc
import paged4check as p4
from pagedcheck import encode, make_table

pytestmark = pytest.mark.gpu


def weights(k, q, scale):
    """(weights of one query over keys k [n, d] in float64, bound of their relative error)."""
    s = scale * (k @ q)
    top = np.abs(q).reshape(-1, 32).max(-1)
    left = 2.0 ** -25 * (np.abs(k).reshape(len(k), -1, 32).sum(-1) @ top)
    ds = abs(scale) * (16 * 2.0 ** -24 * (np.abs(k) @ np.abs(q)) + left) + np.abs(s) * 2.0 ** -22 + (s.max() - s) * 2.0 ** -24
    p = np.exp(s - s.max())
    return p / p.sum(), 2 * ds.max() + 14 * 2.0 ** -22 + 2 * (len(k) / 16 + 16) * 2.0 ** -24


def check(gpu, pool, q, table, lens, group, scale):
    """O and masses, all heads' for every key head of its own: group 1 gives every weight by itself."""
    R, Hq, d = q.shape
    room = table.shape[1] * pool.ps
    opts = nc.paged_options(num_seqs=R, num_q_heads=Hq, max_pages=table.shape[1], scale=scale, **pool.options())
    dq, dt, dl, dm = (nc.DeviceBuffer.from_array(x) for x in (q, table, np.asarray(lens, np.int32), np.zeros((R, room), np.float32)))
    do, work = nc.DeviceBuffer(4 * q.size), nc.DeviceBuffer(nc.paged4_workspace_bytes(opts, mass=True))
    work.memset(0)
    bufs = pool.upload()
    nc.paged4_decode(gpu, dq, *bufs, dt, dl, do, work, opts, mass=dm)
    nc.synchronize()
    o, mass = do.download(np.float32, q.size).reshape(q.shape), dm.download(np.float32, R * room).reshape(R, room)
    nc.paged4_decode(gpu, dq, *bufs, dt, dl, do, work, opts)
    nc.synchronize()
    plain = do.download(np.float32, q.size).reshape(q.shape)
    qf, scale, worst = p4.decode_bits(q, pool.dtype), float(np.float32(scale)), 0.0
    for r in range(R):
        want, allowed = np.zeros(room), np.full(room, 1e-30)
        for h in range(Hq):
            k, pos = p4.rows_of(pool, table, lens, r, 0, h // group)
            v, _ = p4.rows_of(pool, table, lens, r, 1, h // group)
            p, rel = weights(k, qf[r, h], scale)
            want[pos] += p
            allowed[pos] += p * rel
            out, bound = p @ v, (p @ np.abs(v)) * (rel + 2.0 ** -22) + 1e-30
            worst = max(worst, np.max(np.abs(o[r, h] - out) / bound), np.max(np.abs(plain[r, h] - out) / bound))
        worst = max(worst, np.max(np.abs(mass[r] - want) / (allowed + Hq * 2.0 ** -24 * want)))
    assert worst <= 1, worst


@pytest.mark.parametrize("dtype,large", [("f16", 64.0), ("f16", 1024.0), ("f16", 30000.0), ("bf16", 64.0), ("bf16", 4096.0), ("bf16", 1e6)])
@pytest.mark.parametrize("d,ps", [(32, 16), (64, 16), (64, 7), (128, 16), (128, 24)])
@pytest.mark.parametrize("kind", ["channel", "group"])
@pytest.mark.parametrize("group", [1, 4, 8, 20])
def test_queries_with_a_large_channel(gpu, dtype, large, d, ps, kind, group):
    """The keys have nothing in that channel, or in its 32, so that scores are the other channels' business."""
    if kind == "group" and d == 32:
        pytest.skip("one group is all there is")
    rng = np.random.default_rng(int(large) + d + ps + group)
    lens, heads = [90, 300], 2
    pages = sum(-(-n // ps) for n in lens) + 1
    pool = p4.Pool4(rng, pages, heads, ps, d, dtype)
    at = d - 5
    page, head, tok = np.meshgrid(np.arange(pages), np.arange(heads), np.arange(ps), indexing="ij")
    x = rng.standard_normal((*page.shape, d))
    if kind == "channel":
        x[..., at] = 0.0
    else:
        x[..., at // 32 * 32:at // 32 * 32 + 32] = 0.0
    pool.put_values(0, page, head, tok, x)
    table = make_table(rng, lens, ps, pages, -(-max(lens) // ps) + 1)
    q = rng.standard_normal((2, heads * group, d))
    q[..., at] = large * np.where(rng.random(q.shape[:2]) < 0.5, -1.0, 1.0)
    check(gpu, pool, encode(q, dtype), table, lens, group, 1 / np.sqrt(d))


@pytest.mark.parametrize("power", [-90, -100, -112, -120])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_very_small_queries(gpu, power, d):
    """bf16 queries near the type's least normal number, over keys that are as large as those are small."""
    rng = np.random.default_rng(-power + d)
    lens, heads, ps = [150], 2, 16
    pool = p4.Pool4(rng, 10, heads, ps, d, "bf16")
    for page in range(10):
        for t in range(ps):
            pool.put_values(0, page, np.arange(heads), t, rng.standard_normal((heads, d)) * 2.0 ** -power)
    table = np.arange(10, dtype=np.int32)[None]
    q = encode(rng.standard_normal((1, heads, d)) * 2.0 ** power, "bf16")
    check(gpu, pool, q, table, lens, 1, 1 / np.sqrt(d))


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_groups_of_a_query_far_apart(gpu, d, dtype):
    """Every 32 channels of a size of their own, and keys whose groups are as much smaller or larger, or of one size."""
    rng = np.random.default_rng(d)
    lens, heads, ps = [200, 70], 2, 16
    for kind in ("even", "against"):
        pool = p4.Pool4(rng, 20, heads, ps, d, dtype)
        sizes = 2.0 ** rng.permutation([-9, -3, 3, 9])[:d // 32].repeat(32)
        for page in range(20):
            for t in range(ps):
                pool.put_values(0, page, np.arange(heads), t, rng.standard_normal((heads, d)) / (sizes if kind == "against" else sizes.max()))
        table = make_table(rng, lens, ps, 20, 13)
        q = encode(rng.standard_normal((2, heads, d)) * sizes, dtype)
        check(gpu, pool, q, table, lens, 1, 1 / np.sqrt(d))


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("at", [0, 31, -1])
def test_a_channel_that_is_not_finite_gives_nan(gpu, d, at):
    """Whichever 32 it stands in, and no other query's outputs."""
    rng = np.random.default_rng(d + at)
    pool = p4.Pool4(rng, 8, 1, 16, d, "f16")
    table = np.arange(8, dtype=np.int32)[None]
    for bad in (np.inf, -np.inf, np.nan):
        x = rng.standard_normal((1, 4, d))
        x[0, 2, at] = bad
        opts = nc.paged_options(num_seqs=1, num_q_heads=4, max_pages=8, **pool.options())
        dq, dt, dl = (nc.DeviceBuffer.from_array(y) for y in (encode(x, "f16"), table, np.array([100], np.int32)))
        do, work = nc.DeviceBuffer(16 * d), nc.DeviceBuffer(nc.paged4_workspace_bytes(opts))
        work.memset(0)
        nc.paged4_decode(gpu, dq, *pool.upload(), dt, dl, do, work, opts)
        nc.synchronize()
        o = do.download(np.float32, 4 * d).reshape(4, d)
        assert np.isnan(o[2]).all() and np.isfinite(o[[0, 1, 3]]).all()
