"""nc_paged_decode_mass on the GPU: O as nc_paged_decode's, and every token's weights added up, against float64."""

import numpy as np
import pytest

import notcute_flash as nc
import paged4check as p4
from pagedcheck import SENTINEL, Pool, View, encode, make_table

pytestmark = pytest.mark.gpu


def _call(gpu, pool, q, table, lens, mass, mass_stride=0, mass_off=0, scale=None):
    R, Hq, d = q.shape
    opts = nc.paged_options(num_seqs=R, num_q_heads=Hq, max_pages=table.shape[1], scale=scale, **pool.options())
    dq, dt, dl = (nc.DeviceBuffer.from_array(x) for x in (q, table, np.asarray(lens, np.int32)))
    do = nc.DeviceBuffer.from_array(np.full((R + 1) * Hq * d, SENTINEL, np.float32))
    dm = nc.DeviceBuffer.from_array(mass)
    k, v = pool.upload()
    work = nc.DeviceBuffer(nc.paged_mass_workspace_bytes(opts))
    work.memset(0)
    nc.paged_decode_mass(gpu, dq, k, v, dt, dl, do, View(dm, 4 * mass_off), work, opts, mass_stride=mass_stride)
    nc.synchronize()
    o = do.download(np.float32, (R + 1) * Hq * d).reshape(R + 1, Hq, d)
    assert (o[R] == SENTINEL).all()
    return o[:R], dm.download(np.float32, mass.size).reshape(mass.shape)


@pytest.mark.parametrize("lens,heads,group,d,ps,layout,dtype", [
    ([1], 1, 1, 16, 16, "hnd", "f16"), ([20, 0, 257], 2, 4, 64, 16, "hnd", "bf16"), ([300, 33], 3, 5, 128, 32, "nhd", "f16"),
    ([700, 1, 64], 2, 3, 32, 7, "hnd", "bf16"), ([1300], 1, 20, 64, 16, "inter", "f16"), ([513], 2, 33, 32, 16, "nhd", "bf16"),
    ([90, 600], 1, 70, 16, 5, "hnd", "f16"), ([5000], 2, 1, 128, 64, "nhd", "bf16"), ([40] * 300, 4, 2, 64, 16, "hnd", "f16"),
])
def test_mass_matches_float64(gpu, lens, heads, group, d, ps, layout, dtype):
    rng = np.random.default_rng(sum(lens) + d)
    R, width = len(lens), -(-max(lens) // ps) + 1
    pages = sum(-(-n // ps) for n in lens) + 1
    pool = Pool(rng, pages, heads, ps, d, dtype, layout)
    table = make_table(rng, lens, ps, pages, width)
    q = encode(rng.standard_normal((R, heads * group, d)), dtype)
    stride = width * ps + 5
    mass = rng.random((R, stride)).astype(np.float32)
    buf = np.concatenate([np.full(3, SENTINEL, np.float32), mass.ravel()])
    want, bound, madd, mbound = p4.ref_attention(q, pool, table, lens, 1 / np.sqrt(d), group, False)
    got, m = _call(gpu, pool, q, table, lens, buf, stride, 3)
    assert (m[:3] == SENTINEL).all()
    m = m[3:].reshape(R, stride)
    assert (np.abs(got - want) <= bound).all()
    for r, n in enumerate(lens):
        assert np.array_equal(m[r, n:], mass[r, n:])
        assert (np.abs(m[r, :n] - (mass[r, :n].astype(float) + madd[r, :n])) <= mbound[r, :n] + 2.0 ** -23 * m[r, :n]).all()
    # nc_paged_decode splits the keys in the same way where its waves take them one head at a time
    sums = madd.sum(1)
    assert np.allclose(sums, [heads * group if n else 0 for n in lens])


def test_mass_of_absent_keys_sharp_scores_and_nan(gpu):
    rng = np.random.default_rng(4)
    d, ps, heads, group = 64, 16, 2, 2
    pool = Pool(rng, 12, heads, ps, d, "f16")
    table = np.arange(12, dtype=np.int32).reshape(4, 3)
    table[0, 1], table[1] = -1, 99
    lens = [48, 40, 48, 33]
    q = encode(30.0 * rng.standard_normal((4, heads * group, d)), "f16")
    pool.put(0, int(table[3, 0]), 1, 2, encode(np.full(d, np.nan), "f16"))
    mass = np.ones((4, 48), np.float32)
    want, bound, madd, mbound = p4.ref_attention(q[:3], pool, table[:3], lens[:3], 1 / np.sqrt(d), group, False)
    got, m = _call(gpu, pool, q, table, lens, mass)
    assert (np.abs(got[:3] - want) <= bound).all()
    assert (np.abs(m[:3] - (1 + madd)) <= mbound + 2.0 ** -23 * m[:3]).all()
    assert (m[0, 16:32] == 1).all() and (m[1] == 1).all()
    # one head's scores are NaN: so is what the request's tokens gain
    assert np.isnan(m[3, :33]).all() and (m[3, 33:] == 1).all() and np.isnan(got[3, 2:]).all() and np.isfinite(got[3, :2]).all()


def test_steps_add_up_in_a_replayed_graph(gpu):
    """A captured step, replayed with eager calls between: every replay adds the same weights again."""
    rng = np.random.default_rng(6)
    lens, heads, group, d, ps = [400, 0, 70], 2, 4, 64, 16
    pool = Pool(rng, 32, heads, ps, d, "bf16")
    table = make_table(rng, lens, ps, 32, 26)
    q = encode(rng.standard_normal((3, heads * group, d)), "bf16")
    opts = nc.paged_options(num_seqs=3, num_q_heads=heads * group, max_pages=26, **pool.options())
    zero = np.zeros((3, 26 * ps), np.float32)
    dq, dt, dl, dm, dm2 = (nc.DeviceBuffer.from_array(x) for x in (q, table, np.asarray(lens, np.int32), zero, zero))
    do, do2 = nc.DeviceBuffer(q.size * 4), nc.DeviceBuffer(q.size * 4)
    k, v = pool.upload()
    works = []
    for _ in range(2):
        works.append(nc.DeviceBuffer(nc.paged_mass_workspace_bytes(opts)))
        works[-1].memset(0)
    stream = nc.Stream()
    graph = nc.Graph.capture(stream, lambda: nc.paged_decode_mass(gpu, dq, k, v, dt, dl, do, dm, works[0], opts, stream.handle))
    eager = []
    for i in range(4):
        graph.launch(stream)
        stream.synchronize()
        nc.paged_decode_mass(gpu, dq, k, v, dt, dl, do2, dm2, works[1], opts)
        nc.synchronize()
        a, b = (x.download(np.float32, zero.size) for x in (dm, dm2))
        assert np.array_equal(a, b) and np.array_equal(do.download(np.float32, q.size), do2.download(np.float32, q.size))
        eager.append(a)
    graph.destroy()
    assert np.allclose(eager[3], 4 * eager[0].astype(float), rtol=1e-6) and np.isclose(eager[0].sum(), 16, rtol=1e-5)
