"""What the bounds of the 4-bit attention's tests can tell apart, on the CPU: the oracle with the lost bits that they are there for."""

import numpy as np
import pytest

import paged4check as p4
import test_paged4_mass_gpu as tm
import test_paged4_query_gpu as tq
from pagedcheck import decode_bits, encode


def bf16(x):
    return decode_bits(encode(x, "bf16"), "bf16")


@pytest.mark.parametrize("d", [32, 64, 128])
def test_weights_of_two_parts_are_outside_the_bound(d):
    rng = np.random.default_rng(d + 1)
    pool = tm.one_hot(rng, d, d, "f16")
    k, _ = p4.rows_of(pool, np.arange(d // 16)[None], [d], 0, 0, 0)
    s = rng.uniform(0.02, 0.058) * k[:, 9]
    w = np.exp2((s - s.max()) * np.log2(np.e)).astype(np.float32).astype(float)
    parts, left = [], w
    for _ in range(3):
        parts.append(bf16(left))
        left = left - parts[-1]
    p = w / w.sum()
    assert np.max(np.abs((parts[0] + parts[1]) / w.sum() / p - 1)) > tm.ONE_HOT
    assert np.max(np.abs(sum(parts) / w.sum() / p - 1)) < tm.ONE_HOT / 10


@pytest.mark.parametrize("dtype,large", [("f16", 256.0), ("f16", 1024.0), ("bf16", 1024.0), ("bf16", 4096.0)])
def test_queries_rounded_by_their_largest_value_are_outside_the_bound(dtype, large):
    """Every value to 2^-19 of the query's largest, as three parts under one scale would hold it."""
    rng = np.random.default_rng(int(large))
    d, n = 128, 300
    k = rng.standard_normal((n, d))
    q = rng.standard_normal(d)
    k[:, 96:], q[d - 5] = 0.0, large
    q = decode_bits(encode(q, dtype), dtype)
    step = 2.0 ** (np.floor(np.log2(np.abs(q).max())) - 19)
    scale = 1 / np.sqrt(d)
    want, rel = tq.weights(k, q, scale)
    have, _ = tq.weights(k, np.round(q / step) * step, scale)
    assert np.max(np.abs(have / want - 1)) > rel
