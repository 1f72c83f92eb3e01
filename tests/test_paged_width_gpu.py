"""The attention goes by the requests' lengths and not by how wide their block table is: a program keeps a table as wide as
its longest context, and the same requests in it give the same bits."""

import numpy as np
import pytest

import notcute_flash as nc
import pagedcheck as pc

pytestmark = pytest.mark.gpu


def dev(x):
    return nc.DeviceBuffer.from_array(np.ascontiguousarray(x))


@pytest.mark.parametrize("heads,group,d,ps,layout,dtype,lens", [
    # short requests, whose heads take a workgroup's waves in turn
    (8, 1, 32, 16, "nhd", "f16", [200, 200]), (8, 1, 16, 16, "nhd", "bf16", [300, 0, 17, 512]),
    (4, 2, 16, 1, "hnd", "f16", [257, 5]), (8, 4, 64, 16, "nhd", "f16", [200, 31, 512]),
    (4, 3, 64, 1, "hnd", "bf16", [129, 0, 400]), (8, 4, 128, 16, "nhd", "bf16", [400, 100]),
    (4, 1, 128, 24, "nhd", "f16", [511, 33]), (4, 2, 32, 7, "inter", "bf16", [500, 64]),
    # as many as leave a workgroup several heads
    (32, 1, 64, 16, "nhd", "f16", [1 + 5 * i for i in range(20)]), (16, 1, 32, 16, "nhd", "bf16", [1 + 7 * i % 90 for i in range(70)]),
    (8, 2, 16, 5, "nhd", "f16", [1 + 11 * i % 130 for i in range(140)]), (24, 2, 128, 10, "nhd", "bf16", [40 + i for i in range(30)]),
    # one that is long
    (8, 1, 32, 16, "nhd", "f16", [513, 200]), (8, 4, 64, 64, "nhd", "bf16", [9000, 0, 3]),
    (4, 4, 128, 16, "nhd", "f16", [2000, 700]), (8, 2, 16, 1, "hnd", "bf16", [3000, 1]),
    # head-major, and more query heads than neighbouring heads are taken for
    (4, 2, 64, 16, "hnd", "f16", [300, 1000]), (2, 20, 64, 16, "nhd", "bf16", [300, 700])])
def test_tables_of_any_width_give_the_same_bits(gpu, heads, group, d, ps, layout, dtype, lens):
    rng = np.random.default_rng(heads + group + d + ps + len(lens))
    held = [-(-n // ps) for n in lens]
    pool = pc.Pool(rng, sum(held) + 2, heads, ps, d, dtype, layout)
    q = pc.encode(rng.standard_normal((len(lens), heads * group, d)), dtype)
    narrow = pc.make_table(rng, lens, ps, sum(held) + 2, max(held))
    k, v = pool.upload()
    dq, dl = dev(q), dev(np.array(lens, np.int32))
    out = []
    for tokens in (0, 513, 1024, 4096, 20000, 131072):
        width = max(max(held), -(-tokens // ps))
        table = np.full((len(lens), width), 0x7FFFFFFF, dtype=np.int32)
        table[:, :max(held)] = narrow
        opts = nc.paged_options(num_seqs=len(lens), num_q_heads=heads * group, max_pages=width, **pool.options())
        o = nc.DeviceBuffer(4 * q.size)
        nc.paged_decode(gpu, dq, k, v, dev(table), dl, o, nc.paged_workspace(opts), opts)
        nc.synchronize()
        out.append(o.download(np.float32, q.size).reshape(q.shape))
    ref, bound = pc.ref_decode(q, pool, narrow, lens, opts.scale, group)
    assert np.all(np.abs(out[0] - ref) <= bound)
    for x in out[1:]:
        assert np.array_equal(x.view(np.uint32), out[0].view(np.uint32))
