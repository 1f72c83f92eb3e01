"""The 4-bit attention with masses on the GPU over all its ways of cutting the work: short and long requests, many short heads (a wave
each), neighbouring heads in twos and fours, column groups, more than 16 query heads, joins in one round and in several. O and masses
against float64.

Bounds, beside those of a score (test_paged4_query_gpu.py: 16 2^-24 sum |q_i k_i|, 2^-25 of the largest of 32 by Q's parts, 2^-22 of the
score's own size): 2^-22 for every exponential, of which a weight has its own, the sum's and at most 12 that rescale; (n / 16 + 16) 2^-24
for the sums of O and of the weights, of which every lane and product takes a sixteenth; 2^-22 for the quotient. Nothing is left over for
weights that are rounded: three bf16 parts hold 24 bits. A mass adds (Hq / 4 + 4) 2^-24 for the heads' sum and 2^-24 of what it
becomes."""

import numpy as np
import pytest

import notcute_flash as nc
import paged4check as p4
from pagedcheck import SENTINEL, View, decode_bits, encode, make_table
from test_paged4_gpu import SHAPES

pytestmark = pytest.mark.gpu


def reference(q, pool, table, lens, scale, group):
    """(o, its bound, masses added, their bound) in float64."""
    R, Hq, d = q.shape
    room = table.shape[1] * pool.ps
    o, ob, mass, mb = np.zeros((R, Hq, d)), np.zeros((R, Hq, d)), np.zeros((R, room)), np.zeros((R, room))
    qf, scale = decode_bits(q, pool.dtype), float(np.float32(scale))
    for r in range(R):
        for h in range(pool.heads):
            k, pos = p4.rows_of(pool, table, lens, r, 0, h)
            v, _ = p4.rows_of(pool, table, lens, r, 1, h)
            if len(pos) == 0:
                continue
            x = qf[r, h * group:(h + 1) * group]
            s = scale * (x @ k.T)
            gap = s.max(1, keepdims=True) - s
            p = np.exp(-gap)
            p /= p.sum(1, keepdims=True)
            left = np.abs(x).reshape(group, -1, 32).max(-1) @ np.abs(k).reshape(len(k), -1, 32).sum(-1).T
            ds = abs(scale) * 2.0 ** -24 * (16 * (np.abs(x) @ np.abs(k).T) + left / 2) + np.abs(s) * 2.0 ** -22 + gap * 2.0 ** -24
            # by the error of a key's own score and, through the sum, of the others'
            others = (p * ds).sum(1, keepdims=True)
            rest = 14 * 2.0 ** -22 + 2 * (len(pos) / 16 + 16) * 2.0 ** -24
            rel = ds + others + rest
            o[r, h * group:(h + 1) * group] = p @ v
            ob[r, h * group:(h + 1) * group] = (p * rel) @ np.abs(v) + np.abs(p @ v) * 2.0 ** -22
            mass[r, pos] += p.sum(0)
            mb[r, pos] += (p * (rel + 2.0 ** -22 + (Hq / 4 + 4) * 2.0 ** -24)).sum(0)
    return o, ob + 1e-30, mass, mb + 1e-30


def decode(gpu, pool, q, table, lens, mass, stride, off=0, stream=None):
    """(o with a mass, o without one, masses), sentinels checked."""
    R, Hq, d = q.shape
    opts = nc.paged_options(num_seqs=R, num_q_heads=Hq, max_pages=table.shape[1], **pool.options())
    bufs = pool.upload()
    dq, dt, dl, dm = (nc.DeviceBuffer.from_array(x) for x in (q, table, np.asarray(lens, np.int32), mass))
    work = nc.DeviceBuffer(nc.paged4_workspace_bytes(opts, mass=True))
    work.memset(0)
    out = []
    for m in (View(dm, 4 * off), None):
        do = nc.DeviceBuffer.from_array(np.full((R + 1) * Hq * d, SENTINEL, np.float32))
        nc.paged4_decode(gpu, dq, *bufs, dt, dl, do, work, opts, stream, mass=m, mass_stride=stride if m else 0)
        nc.synchronize()
        o = do.download(np.float32, (R + 1) * Hq * d).reshape(R + 1, Hq, d)
        assert (o[R] == SENTINEL).all()
        out.append(o[:R])
    assert not work.download(np.uint32, 5 * 2 * 1024).any()
    return *out, dm.download(np.float32, mass.size)


# SHAPES but its last three, whose rule (5 to 8 query heads a key head, from so many keys on) short requests meet too.
WIDE = [([20] * 130 + [600], 8, 7, 32, 16, "nhd", "f16"), ([30, 0, 600] * 45, 8, 8, 64, 16, "nhd", "bf16"), ([20] * 160 + [515], 4, 5, 128, 40, "nhd", "f16"),
        ([64] * 600, 4, 8, 128, 16, "nhd", "bf16"), ([3, 130] * 300, 2, 16, 32, 16, "hnd", "f16"), ([50] * 520, 2, 3, 64, 9, "nhd", "f16")]


@pytest.mark.parametrize("lens,heads,group,d,ps,layout,dtype", SHAPES[:25] + WIDE)
def test_decode_with_masses_matches_float64(gpu, lens, heads, group, d, ps, layout, dtype):
    rng = np.random.default_rng(len(lens) + d + ps + group)
    R, width = len(lens), -(-max(lens) // ps) + 1
    pages = sum(-(-n // ps) for n in lens) + 1
    pool = p4.Pool4(rng, pages, heads, ps, d, dtype, layout, pad=32 if layout == "inter" else 0)
    table = make_table(rng, lens, ps, pages, width)
    q = encode(rng.standard_normal((R, heads * group, d)), dtype)
    stride = width * ps + 5
    mass = rng.random((R, stride)).astype(np.float32)
    buf = np.concatenate([np.full(3, SENTINEL, np.float32), mass.ravel()])
    want, bound, madd, mbound = reference(q, pool, table, lens, 1 / np.sqrt(d), group)
    with_mass, without, m = decode(gpu, pool, q, table, lens, buf, stride, 3)
    for got in (with_mass, without):
        assert (np.abs(got - want) <= bound).all(), np.max(np.abs(got - want) / bound)
    assert (m[:3] == SENTINEL).all()
    m = m[3:].reshape(R, stride)
    room = width * ps
    off = np.abs(m[:, :room] - (mass[:, :room].astype(float) + madd)) / (mbound + 2.0 ** -24 * m[:, :room])
    for r, n in enumerate(lens):
        assert np.array_equal(m[r, n:], mass[r, n:])
        assert (off[r, :n] <= 1).all(), (r, off[r, :n].max())


def one_hot(rng, d, n, dtype):
    """n <= d keys whose scores under q are exact sums (one channel, a step's bits), V of key j 1 in dim j: O is the weights."""
    pool = p4.Pool4(rng, n // 16, 1, 16, d, dtype)
    level = rng.choice([0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], n) * rng.choice([-1.0, 1.0], n)
    for t in range(n):
        k, v = np.zeros(d), np.zeros(d)
        k[9], v[t] = level[t], 1.0
        pool.put_values(0, t // 16, 0, t % 16, k)
        pool.put_values(1, t // 16, 0, t % 16, v)
    return pool


# A weight's error where its score is exact and at most 0.35 by size: the scaled score and its difference to the maximum 3 2^-24 of
# at most 0.7, two exponentials of an ulp 2 2^-23, 16 additions of the sum 16 2^-24, the quotient's two 2^-23 + 2^-24.
ONE_HOT = 3 * 0.7 * 2.0 ** -24 + 2 * 2.0 ** -23 + 16 * 2.0 ** -24 + 3 * 2.0 ** -24


@pytest.mark.parametrize("group", [1, 4, 8, 16, 17])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_weights_have_f32s_bits(gpu, dtype, d, group):
    """Two bf16 parts of a weight leave up to 2^-18 of it, more than the bound; three leave nothing."""
    rng = np.random.default_rng(d + group)
    pool = one_hot(rng, d, d, dtype)
    table = np.arange(d // 16, dtype=np.int32)[None]
    x = np.zeros((1, group, d))
    x[..., 9] = rng.uniform(0.02, 0.058, (1, group)) * np.sqrt(d)
    q = encode(x, dtype)
    qf, scale = decode_bits(q, dtype), float(np.float32(1 / np.sqrt(d)))
    k, _ = p4.rows_of(pool, table, [d], 0, 0, 0)
    s = scale * (qf[0] @ k.T)
    assert np.abs(s).max() <= 0.35
    p = np.exp(s) / np.exp(s).sum(1, keepdims=True)
    with_mass, without, m = decode(gpu, pool, q, table, [d], np.zeros((1, d), np.float32), 0)
    for got in (with_mass[0], without[0]):
        assert np.max(np.abs(got / p - 1)) <= ONE_HOT, np.max(np.abs(got / p - 1))
    assert np.max(np.abs(m / p.sum(0) - 1)) <= ONE_HOT + (group / 4 + 4) * 2.0 ** -24
