"""The smaller paged cache's operators together, as a serving program runs them: tables and slots (nc_paged_build), rows in, attention
that adds the weights up, eviction, and on; eagerly, captured, from two threads, and with pages far into large pools."""

import threading

import numpy as np
import pytest

import notcute_flash as nc
import paged4check as p4
from pagedcheck import View, encode

pytestmark = pytest.mark.gpu


def dev(x):
    return nc.DeviceBuffer.from_array(np.ascontiguousarray(x))


class Steps:
    """A batch's cache, tables and masses, and every request's rows by themselves."""

    def __init__(self, seed, four, d=64, ps=16, heads=2, group=3, dtype="f16", requests=5, width=20, pages=80, rules=(120, 70, 4, 20)):
        self.rng = np.random.default_rng(seed)
        self.four, self.d, self.ps, self.heads, self.group, self.dtype, self.R = four, d, ps, heads, group, dtype, requests
        self.width, self.pages, self.rules = width, pages, rules
        self.opts = nc.paged_options(num_seqs=requests, num_q_heads=heads * group, num_kv_heads=heads, head_dim=d, page_size=ps, num_pages=pages,
                                     max_pages=width, dtype=dtype)
        values = pages * heads * ps * d
        sizes = (values // 2, values // 2, values // 32, values // 32) if four else (2 * values, 2 * values)
        self.cache = [nc.DeviceBuffer(n) for n in sizes]
        for c in self.cache:
            c.memset(0)
        self.table, self.lens = dev(np.full((requests, width), -1, np.int32)), dev(np.zeros(requests, np.int32))
        self.free, self.counts = dev(self.rng.permutation(pages).astype(np.int32)), dev(np.zeros(4, np.int32))
        self.mass = dev(np.zeros((requests, width * ps), np.float32))
        self.off, self.dnew = nc.DeviceBuffer(4 * requests + 4), nc.DeviceBuffer(4 * requests)
        need = nc.paged4_workspace_bytes(self.opts, mass=True) if four else nc.paged_mass_workspace_bytes(self.opts)
        self.work, self.ework = nc.DeviceBuffer(need), nc.DeviceBuffer(nc.paged_evict_workspace_bytes(self.opts))
        self.work.memset(0)
        self.history = [[] for _ in range(requests)]
        self.places = 0

    def prepare(self, new, places):
        """The step's new rows and queries; the slot map has room for `places` rows."""
        new, row = np.asarray(new, np.int32), (places, self.heads, self.d)
        self.q = encode(self.rng.standard_normal((self.R, self.heads * self.group, self.d)), self.dtype)
        rows = [encode(self.rng.standard_normal(row), self.dtype) for _ in "kv"]
        if self.places != places:
            self.places, self.slots = places, nc.DeviceBuffer(4 * places)
            self.dk, self.dv = (nc.DeviceBuffer(rows[0].nbytes) for _ in "kv")
            self.dq, self.do = nc.DeviceBuffer(self.q.nbytes), nc.DeviceBuffer(2 * self.q.nbytes)
        for buf, x in ((self.dnew, new), (self.dk, rows[0]), (self.dv, rows[1]), (self.dq, self.q)):
            buf.upload(x)
        values = [p4.decode_bits(x, self.dtype) for x in rows]
        if self.four:
            values = [p4.values(*p4.quantise(x, self.dtype)) for x in values]
        at = 0
        for h, n in zip(self.history, new):
            h += [(values[0][at + i], values[1][at + i]) for i in range(n)]
            at += n

    def attend(self, gpu, stream=None):
        nc.paged_build(gpu, self.lens, self.dnew, self.free, View(self.counts, 0, 4), self.table, self.lens, self.off, self.slots, self.counts,
                       self.opts, stream)
        if self.four:
            nc.paged4_append(gpu, self.dk, self.dv, self.slots, *self.cache, self.opts, stream)
            nc.paged4_decode(gpu, self.dq, *self.cache, self.table, self.lens, self.do, self.work, self.opts, stream, mass=self.mass)
        else:
            nc.paged_append(gpu, self.dk, self.dv, self.slots, *self.cache, self.opts, stream)
            nc.paged_decode_mass(gpu, self.dq, *self.cache, self.table, self.lens, self.do, self.mass, self.work, self.opts, stream)

    def evict(self, gpu, stream=None):
        f = nc.paged4_evict if self.four else nc.paged_evict
        f(gpu, self.table, self.lens, self.mass, *self.cache, self.free, View(self.counts, 0, 4), self.lens, self.counts, self.ework,
          nc.evict_rules(**dict(zip(("limit", "budget", "sinks", "recent"), self.rules))), self.opts, stream)

    def lists(self):
        return (self.lens.download(np.int32, self.R), self.mass.download(np.float32, self.R * self.width * self.ps).reshape(self.R, -1),
                self.table.download(np.int32, self.R * self.width).reshape(self.R, -1), self.free.download(np.int32, self.pages),
                self.counts.download(np.int32, 4))

    def verify(self, before, what):
        """O, and the masses against those `before` the step."""
        lens, mass, _, _, counts = self.lists()
        assert lens.tolist() == [len(h) for h in self.history] and counts[3] == 0, what
        out = self.do.download(np.float32, self.q.size).reshape(self.q.shape)
        for r, h in enumerate(self.history):
            n = max(len(h), 1)
            pool = _Rows(h, self.heads, self.d, self.dtype)
            want, bound, add, abound = p4.ref_attention(self.q[r:r + 1], pool, np.zeros((1, 1), np.int32), [len(h)], self.opts.scale, self.group,
                                                        self.four)
            assert (np.abs(out[r] - want[0]) <= bound[0]).all(), (what, r)
            gained = mass[r, :n].astype(float) - before[r, :n] - add[0, :n]
            assert (np.abs(gained) <= abound[0, :n] + 2.0 ** -23 * np.abs(mass[r, :n])).all(), (what, r)
        return mass

    def verify_evict(self, gpu, what):
        lens, mass, table, free, counts = self.lists()
        kept, out, m, f, c = p4.ref_evict(lens, mass, table, free, counts[0], self.ps, self.width * self.ps, self.rules)
        self.evict(gpu)
        nc.synchronize()
        got = self.lists()
        assert got[0].tolist() == out.tolist() and np.array_equal(got[1], m) and np.array_equal(got[3], f) and np.array_equal(got[4], c), what
        for r, keep in enumerate(kept):
            if keep is not None:
                self.history[r] = [self.history[r][j] for j in keep]
        return int(c[1])

    def state(self):
        return [x.download(np.uint8, x.nbytes) for x in (self.do, self.mass, self.lens, self.table, self.counts, self.free, *self.cache)]


class _Rows:
    """Values of one request as a pool of one page."""

    def __init__(self, history, heads, d, dtype):
        self.pages, self.heads, self.d, self.dtype, self.ps = 1, heads, d, dtype, max(len(history), 1)
        self.x = [np.array([row[i] for row in history]).reshape(-1, heads, d) for i in range(2)]

    def get(self, which, page, head, tok):
        return self.x[which][tok, head]


CASES = [(True, 64, 16, 2, 3, "f16"), (True, 128, 7, 1, 8, "bf16"), (True, 32, 16, 4, 12, "f16"), (False, 64, 16, 2, 3, "bf16"), (False, 16, 9, 3, 2, "f16")]


@pytest.mark.parametrize("four,d,ps,heads,group,dtype", CASES)
def test_steps_together(gpu, four, d, ps, heads, group, dtype):
    s = Steps(d + ps, four, d, ps, heads, group, dtype, width=-(-200 // ps), pages=-(-700 // ps))
    before, cut = s.lists()[1], 0
    for step, new in enumerate(([110, 0, 130, 1, 60], [1, 1, 1, 0, 1], [20, 1, 1, 1, 90], [1, 0, 70, 1, 1], [60, 1, 1, 3, 1], [1, 1, 1, 1, 1])):
        s.prepare(new, 320)
        s.attend(gpu)
        nc.synchronize()
        s.verify(before, f"step {step}")
        cut += s.verify_evict(gpu, f"eviction {step}")
        before = s.lists()[1]
    assert cut >= 4


@pytest.mark.parametrize("four", [True, False])
def test_captured_steps_replay_as_eager_ones(gpu, four):
    """A step with its eviction, first launched under capture through a module of its own, and replayed; its twin runs eagerly
    between the replays, and every buffer of the two is the same."""
    module = nc.Module.load_embedded()
    kw = dict(ps=7, width=30, pages=110) if four else {}
    a, b = Steps(31, four, **kw), Steps(31, four, **kw)
    stream = nc.Stream()
    graph = None
    try:
        for step in range(12):
            new = [100, 0, 130, 1, 60] if step == 0 else [int(step % 4 != r % 4) * (1 + 40 * int(step == 6 and r < 2)) for r in range(5)]
            for s in (a, b):
                s.prepare(new, 300)
            if graph is None:
                graph = nc.Graph.capture(stream, lambda: (a.attend(module, stream.handle), a.evict(module, stream.handle)))
            graph.launch(stream)
            b.attend(gpu)
            b.evict(gpu)
            nc.synchronize()
            stream.synchronize()
            for i, (x, y) in enumerate(zip(a.state(), b.state())):
                assert np.array_equal(x, y), (step, i)
    finally:
        if graph is not None:
            graph.destroy()
        stream.destroy()
        module.unload()


def test_two_threads_launch_through_one_module(gpu):
    """Two host threads at once, each with a stream, buffers and workspaces of its own."""
    module = nc.Module.load_embedded()
    sides = [Steps(41, True), Steps(42, False)]
    alone = [Steps(41, True), Steps(42, False)]
    streams = [nc.Stream() for _ in sides]
    plan = ([100, 0, 130, 1, 60], [1, 1, 1, 0, 1], [40, 1, 1, 1, 70], [1, 1, 1, 1, 1])
    errors = []

    def steps(s, handle, wait):
        for new in plan:
            s.prepare(new, 300)
            s.attend(module, handle)
            s.evict(module, handle)
            wait()

    def guarded(*x):
        try:
            steps(*x)
        except BaseException as e:  # shown by the main thread
            errors.append(e)

    threads = [threading.Thread(target=guarded, args=(s, st.handle, st.synchronize)) for s, st in zip(sides, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for s in alone:
        steps(s, None, nc.synchronize)
    for s, t in zip(sides, alone):
        for x, y in zip(s.state(), t.state()):
            assert np.array_equal(x, y)
    for st in streams:
        st.destroy()
    module.unload()


def test_a_prompt_goes_on_behind_a_cached_one(gpu):
    """Cached rows are read back as dense ones, the flash forward takes them with the prompt's own, and its last row is what the
    decode over the cache gives."""
    rng = np.random.default_rng(5)
    S, old, heads, d, ps = 90, 50, 4, 64, 16
    pages = -(-S // ps)
    opts = nc.paged_options(num_q_heads=heads, head_dim=d, page_size=ps, num_pages=pages, max_pages=pages)
    values = pages * heads * ps * d
    cache = [nc.DeviceBuffer(n) for n in (values // 2, values // 2, values // 32, values // 32)]
    for c in cache:
        c.memset(0)
    order = rng.permutation(pages).astype(np.int32)
    slots = (order[np.arange(S) // ps] * ps + np.arange(S) % ps).astype(np.int32)
    rows = [encode(rng.standard_normal((S, heads, d)), "f16") for _ in "kv"]
    for part in (slice(0, old), slice(old, S)):
        nc.paged4_append(gpu, dev(rows[0][part]), dev(rows[1][part]), dev(slots[part]), *cache, opts)
    # dense [head][token][dim]: a row's heads stand S*d apart
    back = nc.PagedOptions.from_buffer_copy(opts)
    back.row_stride, back.row_head_stride = d, S * d
    dk, dv = (nc.DeviceBuffer(heads * S * d * 2) for _ in "kv")
    nc.paged4_read(gpu, *cache, dev(slots), dk, dv, back)
    q = encode(rng.standard_normal((heads, S, d)), "f16")
    do, dq = nc.DeviceBuffer(heads * S * d * 4), dev(q)
    nc.flash_launch(gpu, dq, dk, dv, do, nc.options(seq_len=S, head_dim=d, batch_heads=heads, causal=True))
    work = nc.DeviceBuffer(nc.paged4_workspace_bytes(opts))
    work.memset(0)
    one = nc.PagedOptions.from_buffer_copy(opts)
    one.q_head_stride, one.q_stride = S * d, heads * S * d
    out = nc.DeviceBuffer(heads * d * 4)
    nc.paged4_decode(gpu, View(dq, 2 * (S - 1) * d), *cache, dev(order[None]), dev(np.array([S], np.int32)), out, work, one)
    nc.synchronize()
    import flashcheck as fc

    last = do.download(np.float32, heads * S * d).reshape(heads, S, d)[:, -1]
    assert np.max(np.abs(out.download(np.float32, heads * d).reshape(heads, d) - last)) <= fc.MAX_ABS


@pytest.mark.parametrize("pages,page_size", [(262144 - 8, 16), (262144 + 9, 16), (400000, 13)])
def test_pages_far_into_large_pools(gpu, pages, page_size):
    """Pools of about and of more than 2^32 values, the pages at both ends of them: rows, attention, masses and eviction."""
    rng = np.random.default_rng(pages)
    heads, d, n = 8, 128, 5 * page_size + 3
    values = pages * heads * page_size * d
    cache = [nc.DeviceBuffer(x) for x in (values // 2, values // 2, values // 32, values // 32)]
    try:
        for c in cache:
            c.memset(0xFF)  # scales of NaN
        table = np.array([[0, pages - 1, pages // 2, 1, pages - 2, pages - 3]], np.int32)
        width = table.shape[1]
        opts = nc.paged_options(num_q_heads=2 * heads, num_kv_heads=heads, head_dim=d, page_size=page_size, num_pages=pages, max_pages=width,
                                dtype="bf16")
        at = np.arange(n)
        slots = (table[0, at // page_size].astype(np.int64) * page_size + at % page_size).astype(np.int32)
        rows = [encode(rng.standard_normal((n, heads, d)), "bf16") for _ in "kv"]
        nc.paged4_append(gpu, dev(rows[0]), dev(rows[1]), dev(slots), *cache, opts)
        hist = [p4.values(*p4.quantise(p4.decode_bits(x, "bf16"), "bf16")) for x in rows]
        pool = _Rows(list(zip(*hist)), heads, d, "bf16")
        q = encode(rng.standard_normal((1, 2 * heads, d)), "bf16")
        want, bound, add, abound = p4.ref_attention(q, pool, np.zeros((1, 1), np.int32), [n], opts.scale, 2, True)
        work = nc.DeviceBuffer(nc.paged4_workspace_bytes(opts, mass=True))
        work.memset(0)
        out, mass = nc.DeviceBuffer(q.size * 4), dev(np.zeros(width * page_size, np.float32))
        dt, dl = dev(table), dev(np.array([n], np.int32))
        nc.paged4_decode(gpu, dev(q), *cache, dt, dl, out, work, opts, mass=mass)
        nc.synchronize()
        got, m = out.download(np.float32, q.size).reshape(q.shape), mass.download(np.float32, width * page_size)
        assert (np.abs(got - want) <= bound).all() and (np.abs(m[:n] - add[0]) <= abound[0] + 2.0 ** -23 * m[:n]).all()
        keep, counts, work2 = n - 2 * page_size, dev(np.array([6, 0, 0, 0], np.int32)), nc.DeviceBuffer(nc.paged_evict_workspace_bytes(opts))
        free = dev(np.arange(8, dtype=np.int32))
        kept, *_ = p4.ref_evict(np.array([n]), m[None], table, np.arange(8, dtype=np.int32), 6, page_size, width * page_size, (keep, keep, 2, 3))
        nc.paged4_evict(gpu, dt, dl, mass, *cache, free, View(counts, 0, 4), dl, counts, work2, nc.evict_rules(limit=keep, budget=keep, sinks=2, recent=3),
                        opts)
        back = [nc.DeviceBuffer(keep * heads * d * 2) for _ in "kv"]
        nc.paged4_read(gpu, *cache, dev(slots[:keep]), *back, opts)
        nc.synchronize()
        assert dl.download(np.int32, 1)[0] == keep and counts.download(np.int32, 4).tolist() == [4, 1, 2, 2 * page_size]
        for x, b in zip(hist, back):
            assert np.array_equal(p4.decode_bits(b.download(np.uint16, keep * heads * d), "bf16").reshape(keep, heads, d), x[kept[0]])
    finally:
        for c in cache:
            c.free()


def test_harness_command(gpu, capsys):
    """flash_harness.py paged4: a record per case, each within its tolerance."""
    import json

    import flash_harness as fh

    assert fh.main(["paged4", "--warmup", "1", "--iters", "3"]) == 0
    recs = [json.loads(line) for line in capsys.readouterr().out.splitlines() if line.startswith("{")]
    assert len(recs) == len(fh.PAGED4_CASES)
    for r in recs:
        assert set(r) == set(fh.RECORD_KEYS) and r["kernel"] == "paged4_attention"
        assert r["correct"] and r["max_abs_error"] <= fh.PAGED_TOL and r["min_ms"] > 0
