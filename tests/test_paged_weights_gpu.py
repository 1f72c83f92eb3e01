"""The attention's weights one by one: keys whose scores are exact in f32, so that what is left of the error is the
exponential's, the split of the weight into 16-bit parts, the sums' and the quotient's."""

import numpy as np
import pytest

import notcute_flash as nc
import pagedcheck as pc

pytestmark = pytest.mark.gpu

# scale * log2(e) rounds to 1 in f32: a score in bits is the dot product itself.
LN2 = float(np.float32(np.log(2.0)))
# Q's first three dims. K's are integers of 8 bits at most (the third's over 1024), exact in f16 and bf16, and the dot
# product is a multiple of 2^-24.
Q3 = np.array([1.0, 2.0 ** -8, 2.0 ** -14])


def dev(x):
    return nc.DeviceBuffer.from_array(np.ascontiguousarray(x))


def bits_key(rng):
    """K's first three dims for a score between -1 and 0 bits, to the last of f32's 24."""
    return -np.array([0, rng.integers(1, 255), rng.integers(0, 256) / 1024.0])


def attend(gpu, rng, keys, values, d, ps, dtype):
    """O of one request per row of `keys` ([R, n, 3], the first dims of K) and `values` ([R, n]: V, the same in every dim),
    one head."""
    assert np.float32(LN2) * np.float32(1.4426950408889634) == np.float32(1.0)
    R, n, _ = keys.shape
    width = -(-n // ps)
    pool = pc.Pool(rng, R * width, 1, ps, d, dtype, poison=True)
    table = rng.permutation(R * width).reshape(R, width).astype(np.int32)
    k, v = np.zeros((n, d)), np.zeros((n, d))
    at = np.arange(n)
    for r in range(R):
        k[:, :3] = keys[r]
        v[:] = values[r][:, None]
        for which, x in ((0, k), (1, v)):
            bits = pc.encode(x, dtype)
            assert np.array_equal(pc.decode_bits(bits, dtype), x)
            pool.put(which, table[r, at // ps], 0, at % ps, bits)
    q = np.zeros((R, 1, d))
    q[:, 0, :3] = Q3
    opts = nc.paged_options(num_seqs=R, max_pages=width, scale=LN2, num_q_heads=1, **pool.options())
    kc, vc = pool.upload()
    o = nc.DeviceBuffer(4 * R * d)
    nc.paged_decode(gpu, dev(pc.encode(q, dtype)), kc, vc, dev(table), dev(np.full(R, n, np.int32)), o,
                    nc.paged_workspace(opts), opts)
    nc.synchronize()
    return o.download(np.float32, R * d).reshape(R, d).astype(np.float64)


def weights(keys):
    """exp(scale * score) in float64."""
    return np.exp(LN2 * (keys @ Q3))


@pytest.mark.parametrize("d,ps,dtype", [(16, 16, "bf16"), (32, 7, "bf16"), (64, 16, "bf16"), (128, 16, "bf16"), (128, 5, "bf16"),
                                        (16, 16, "f16"), (64, 16, "f16"), (64, 3, "f16"), (128, 16, "f16")])
def test_one_weight_beside_the_largest(gpu, d, ps, dtype):
    """15 keys of the largest score and V = 0, and a last one less than a bit below with V = 1: O = w / (15 + w).

    In units of 2^-24: the exponential 2 (an ulp); the parts' sum 4 in f16 (2^-22), 1 in bf16; each of the three products
    that add the parts up 2 (an ulp); the sum of the weights 3 (one addition in the lane that has w last and two over the
    lanes; the 1s are exact); the reciprocal 2 and the product with it 1; log2(e), scale * log2(e) and the score's product
    with it 1 each, times the score of at most ln 2. Together less than 21 in f16 and 18 in bf16."""
    rng = np.random.default_rng(d + ps)
    R, n = 400, 16
    keys, values = np.zeros((R, n, 3)), np.zeros((R, n))
    for r in range(R):
        keys[r, -1] = bits_key(rng)
    values[:, -1] = 1.0
    w = weights(keys[:, -1])
    want = w / (15.0 + w)
    out = attend(gpu, rng, keys, values, d, ps, dtype)
    off = np.abs(out / want[:, None] - 1.0).max() * 2.0 ** 24
    assert off <= {"f16": 4, "bf16": 1}[dtype] + 2 + 6 + 3 + 2 + 1 + 3 * np.log(2.0), f"off by {off:.1f} x 2^-24"


@pytest.mark.parametrize("least,most,dtype", [(16, 24, "f16"), (24, 32, "f16"), (32, 40, "f16"), (20, 45, "bf16"), (45, 70, "bf16")])
@pytest.mark.parametrize("d,ps", [(16, 16), (32, 7), (64, 16), (64, 5), (128, 16), (128, 3)])
def test_small_weights_where_the_largest_counts_for_nothing(gpu, d, ps, least, most, dtype):
    """One key of the largest score with V = 0 and 199 keys `least` to `most` bits below it: O is made of theirs alone.

    In units of 2^-24, relative to sum w |v|: the exponential 2, the parts' sum 4 (2^-22), sums over n keys and up to 40
    joins of lanes, waves and pieces 2 each (an ulp), the factors of a larger maximum and of the waves' join 3 each, the
    quotient 3, the score's three roundings times itself (scores are multiples of 2^-8 bits, so their differences are
    exact). Weights of less than 2^-29 (f16) or 2^-70 (bf16) are off by up to 2^-51 or 2^-93 of the largest weight."""
    rng = np.random.default_rng(1000 * d + 100 * ps + most)
    R, n = 40, 200
    keys, values = np.zeros((R, n, 3)), rng.integers(-64, 65, (R, n)) / 16.0
    for r in range(R):
        keys[r, :, 0] = -rng.integers(least, most, n)
        keys[r, :, 1] = -rng.integers(0, 256, n)
        top = 0 if r % 2 else rng.integers(0, n)
        keys[r, top] = values[r, top] = 0.0
    w = weights(keys)
    want = (w * values).sum(1) / w.sum(1)
    out = attend(gpu, rng, keys, values, d, ps, dtype)
    units = 2 + 4 + 2 * (n + 40) + 6 + 3 + 3 * LN2 * (most + 1)
    bound = units * 2.0 ** -24 * (w * np.abs(values)).sum(1) + {"f16": 2.0 ** -51, "bf16": 2.0 ** -93}[dtype] * np.abs(values).sum(1)
    off = (np.abs(out - want[:, None]).max(1) / bound).max()
    assert off <= 1.0, f"off by {off:.2f} bounds"


@pytest.mark.parametrize("n", [1, 40, 700, 20000])
@pytest.mark.parametrize("d,ps,dtype", [(16, 16, "f16"), (64, 16, "bf16"), (64, 7, "f16"), (128, 16, "f16")])
def test_scores_and_values_of_infinity_are_not_hidden(gpu, n, d, ps, dtype):
    """A score of +infinity among the keys that count gives NaN, and an infinite V that infinity: at the first key, the last
    and one between, whichever wave and piece has it."""
    rng = np.random.default_rng(n + d)
    at = sorted({0, n // 3, n - 1})
    keys, values = np.zeros((2 * len(at) + 1, n, 3)), np.ones((2 * len(at) + 1, n))
    keys[:, :, 1] = -rng.integers(0, 256, (2 * len(at) + 1, n))
    for i, j in enumerate(at):
        keys[2 * i, j, 0] = np.inf
        values[2 * i + 1, j] = -np.inf
    out = attend(gpu, rng, keys, values, d, ps, dtype)
    assert np.all(np.isnan(out[:-1:2]))
    assert np.all(out[1:-1:2] == -np.inf)
    assert np.all(np.abs(out[-1] - 1.0) <= (n + 40) * 2.0 ** -23)
