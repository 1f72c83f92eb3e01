"""Batches of which most requests are empty, as a step captured for a fixed number of them has: what the attention of the
others gives, and that it does not wait for the empty ones one by one."""

import numpy as np
import pytest

import notcute_flash as nc
import pagedcheck as pc

pytestmark = pytest.mark.gpu


def dev(x):
    return nc.DeviceBuffer.from_array(np.ascontiguousarray(x))


class Batch:
    """`lens`: request -> length, the others are empty."""

    def __init__(self, count, lens, heads=4, group=2, d=64, ps=16, layout="hnd", dtype="f16", seed=0):
        rng = np.random.default_rng(seed)
        self.lens = np.zeros(count, np.int32)
        for r, n in lens.items():
            self.lens[r] = n
        held = [-(-int(n) // ps) for n in self.lens]
        self.group = group
        self.pool = pc.Pool(rng, sum(held) + 1, heads, ps, d, dtype, layout)
        self.table = pc.make_table(rng, self.lens, ps, sum(held) + 1, max(held), spare=0x7FFFFFFF)
        self.q = pc.encode(rng.standard_normal((count, heads * group, d)), dtype)
        self.opts = nc.paged_options(num_seqs=count, num_q_heads=heads * group, max_pages=max(held), **self.pool.options())
        self.o = dev(np.full(self.q.shape, pc.SENTINEL, np.float32))
        self.args = [dev(self.q), *self.pool.upload(), dev(self.table), dev(self.lens), self.o, nc.paged_workspace(self.opts)]

    def launch(self, module, stream=None):
        nc.paged_decode(module, *self.args, self.opts, stream)

    def check(self):
        out = self.o.download(np.float32, self.q.size).reshape(self.q.shape)
        busy = np.flatnonzero(self.lens)
        ref, bound = pc.ref_decode(self.q[busy], self.pool, self.table[busy], self.lens[busy], self.opts.scale, self.group)
        assert np.all(np.abs(out[busy] - ref) <= bound)
        out[busy] = 0.0
        assert not np.any(out), "an empty request's rows are not zeros"


@pytest.mark.parametrize("count", [2, 64, 65, 66, 129, 130, 200, 700, 4097])
@pytest.mark.parametrize("d,ps,layout,dtype", [(64, 16, "hnd", "f16"), (32, 7, "nhd", "bf16"), (128, 16, "nhd", "bf16"), (16, 16, "hnd", "f16")])
def test_few_of_many(gpu, count, d, ps, layout, dtype):
    """Requests with keys at the ends, around multiples of 64 from one another, next to each other, one or several to a
    workgroup's share, long and short."""
    last = count - 1
    for lens in ({0: 100}, {last: 100}, {0: 33, last: 700}, {0: 1, 1: 1, last // 2: 40, last: 1},
                 {r: 5 + r % 40 for r in range(0, count, 65)}, {r: 300 for r in range(0, count, 64) if r < 700},
                 {0: 3000, last // 3: 20, last: 2}):
        b = Batch(count, lens, d=d, ps=ps, layout=layout, dtype=dtype, seed=count + d)
        b.launch(gpu)
        nc.synchronize()
        b.check()


def test_time_does_not_go_by_the_empty_ones_behind_or_between(gpu):
    """4096 requests of which the first, or the first and the last, have keys take about as long as where the last has them
    (26 us; one empty request after the other took 271): no more than twice as long, each the best of 50 calls."""
    times = []
    for lens in ({4095: 100}, {0: 100}, {0: 100, 4095: 100}):
        b = Batch(4096, lens)
        start, stop, best = nc.Event(), nc.Event(), np.inf
        for _ in range(50):
            start.record()
            for _ in range(4):
                b.launch(gpu)
            stop.record()
            stop.synchronize()
            best = min(best, nc.Event.elapsed(start, stop))
        start.destroy()
        stop.destroy()
        b.check()
        times.append(best)
    assert max(times[1:]) <= 2 * times[0], times
