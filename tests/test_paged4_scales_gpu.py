"""Scale bytes of a 4-bit cache that nc_paged4_append does not write, as another writer of the format may: the least ones, whose values
16-bit types hold as subnormal numbers, and the largest, whose larger values no f32 holds."""

import numpy as np
import pytest

import notcute_flash as nc
import paged4check as p4
from pagedcheck import encode

pytestmark = pytest.mark.gpu


def pool_of(rng, d, dtype, scales, n=64):
    """One head's n tokens with every code and these scale bytes in turn, for K and for V."""
    pool = p4.Pool4(rng, n // 16, 1, 16, d, dtype)
    for which in range(2):
        for t in range(n):
            codes = rng.permutation(np.arange(d) % 16).astype(np.uint8)
            pool.put(which, t // 16, 0, t % 16, codes, np.array([scales[(t + g + which) % len(scales)] for g in range(d // 32)], np.uint8))
    return pool


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("scales", [[0, 1], [0, 1, 2, 3, 255], [95, 100, 101, 102, 103, 104], [139, 140, 141, 142, 143, 150], [250, 251, 252, 253, 254]])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_read_of_every_scale(gpu, dtype, scales, d):
    """Values are exact where the type holds them, else the nearest that it holds, an infinity above the largest."""
    rng = np.random.default_rng(d + scales[0])
    pool = pool_of(rng, d, dtype, scales)
    slots = rng.permutation(64).astype(np.int32)
    o = nc.paged_options(num_q_heads=1, **pool.options())
    dk, dv = nc.DeviceBuffer(64 * d * 2), nc.DeviceBuffer(64 * d * 2)
    nc.paged4_read(gpu, *pool.upload(), nc.DeviceBuffer.from_array(slots), dk, dv, o)
    nc.synchronize()
    for which, b in enumerate((dk, dv)):
        got = p4.decode_bits(b.download(np.uint16, 64 * d).reshape(64, d), dtype)
        x = pool.get(which, slots // 16, 0, slots % 16)
        with np.errstate(over="ignore"):
            want = p4.decode_bits(encode(x, dtype), dtype)
        same = (got == want) | (np.isnan(got) & np.isnan(want))
        assert same.all(), (x[~same][:8], got[~same][:8], want[~same][:8])
        assert (np.signbit(got) == np.signbit(want))[~np.isnan(want)].all()


def attend(gpu, pool, q, n=64):
    opts = nc.paged_options(num_seqs=1, num_q_heads=q.shape[1], max_pages=pool.pages, scale=1.0, **pool.options())
    dq, dt, dl = (nc.DeviceBuffer.from_array(x) for x in (q, np.arange(pool.pages, dtype=np.int32)[None], np.array([n], np.int32)))
    do, dm = nc.DeviceBuffer(4 * q.size), nc.DeviceBuffer.from_array(np.zeros(pool.pages * 16, np.float32))
    work = nc.DeviceBuffer(nc.paged4_workspace_bytes(opts, mass=True))
    work.memset(0)
    nc.paged4_decode(gpu, dq, *pool.upload(), dt, dl, do, work, opts, mass=dm)
    nc.synchronize()
    return do.download(np.float32, q.size).reshape(q.shape), dm.download(np.float32, pool.pages * 16)


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("group", [1, 8, 16])
def test_attention_over_the_least_scales(gpu, d, group):
    """K: scores that are 0 as far as an exponential can tell, so equal weights; V: values below 2^-124, which may count as 0."""
    rng = np.random.default_rng(d + group)
    q = encode(rng.standard_normal((1, group, d)), "bf16")
    pool = pool_of(rng, d, "bf16", [0, 1])
    o, mass = attend(gpu, pool, q)
    assert (np.abs(o) <= 2.0 ** -123).all()
    assert np.allclose(mass, group / 64, rtol=1e-6, atol=0)
    # keys of such scales beside ordinary ones
    k = rng.standard_normal((64, d))
    for t in range(1, 64, 2):
        pool.put_values(0, t // 16, 0, t % 16, k[t])
    for t in range(64):
        pool.put_values(1, t // 16, 0, t % 16, k[t])
    table = np.arange(4, dtype=np.int32)[None]
    want, bound, madd, mbound = p4.ref_attention(q, pool, table, [64], 1.0, group, True)
    o, mass = attend(gpu, pool, q)
    assert (np.abs(o - want) <= bound).all() and (np.abs(mass - madd[0]) <= mbound[0] + 2.0 ** -23 * mass).all()


@pytest.mark.parametrize("d", [32, 64, 128])
def test_attention_over_the_largest_scales(gpu, d):
    """V of scale bytes 253 and 254 as far as bf16 holds the values; keys of such scales under queries as small."""
    rng = np.random.default_rng(d)
    pool = p4.Pool4(rng, 4, 1, 16, d, "bf16")
    for t in range(64):
        codes = rng.integers(0, 3, d).astype(np.uint8) | rng.integers(0, 2, d).astype(np.uint8) << 3  # 0, 0.5, 1
        pool.put(1, t // 16, 0, t % 16, codes, np.full(d // 32, 253 + t % 2, np.uint8))
        pool.put(0, t // 16, 0, t % 16, codes, np.full(d // 32, 253 + t % 2, np.uint8))
    q = encode(rng.standard_normal((1, 4, d)) * 2.0 ** -126, "bf16")
    want, bound, madd, mbound = p4.ref_attention(q, pool, np.arange(4, dtype=np.int32)[None], [64], 1.0, 4, True)
    o, mass = attend(gpu, pool, q)
    assert (np.abs(o - want) <= bound).all(), np.max(np.abs(o - want) / bound)
    assert (np.abs(mass - madd[0]) <= mbound[0] + 2.0 ** -23 * mass).all()


@pytest.mark.parametrize("d", [32, 64, 128])
def test_values_that_f32_does_not_hold(gpu, d):
    """V of 2^128 and more counts as infinite: its dim of O is infinite or NaN, and no other."""
    rng = np.random.default_rng(d)
    pool = p4.Pool4(rng, 4, 1, 16, d, "bf16")
    codes = rng.integers(0, 3, d).astype(np.uint8)
    codes[5] = 7  # 6 2^126
    pool.put(1, 1, 0, 3, codes, np.full(d // 32, 253, np.uint8))
    q = encode(rng.standard_normal((1, 4, d)), "bf16")
    o, mass = attend(gpu, pool, q)
    assert not np.isfinite(o[0, :, 5]).any() and np.isfinite(np.delete(o[0], 5, axis=1)).all()
    assert np.isfinite(mass).all() and abs(mass.sum() - 4) < 1e-5
