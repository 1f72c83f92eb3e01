"""Paged cache, on the CPU: validation and refusals of the C ABI (include/notcute_paged.h), the layout of its
options, and the index arithmetic that the kernels share with the host (csrc/paged_args.h)."""

import ctypes
import os
import re
import subprocess

import numpy as np
import pytest

import notcute_flash as nc
import pagedcheck as pc

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "notcute_paged.h")
CSRC = os.path.join(ROOT, "not-cute-zig_amd", "csrc")
INVALID, OVERFLOW = "InvalidValue", "Overflow"


def good(**kw):
    base = dict(num_seqs=4, num_q_heads=8, num_kv_heads=2, head_dim=64, page_size=16, num_pages=50, max_pages=10)
    base.update(kw)
    return nc.paged_options(**base)


def test_library_exports_every_declared_function():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(nc_paged_[a-z0-9_]+)\s*\(", text)))
    assert len(names) == 6
    for n in names:
        assert hasattr(nc.load_library(), n), n
        assert n in nc._SIGS, n


def test_options_layout_matches_binding(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "notcute_paged.h"', "int main(void) {",
             'printf("- %zu %zu\\n", sizeof(nc_paged_options), _Alignof(nc_paged_options));']
    for f, _ in nc.PagedOptions._fields_:
        lines.append(f'printf("{f} %zu %zu\\n", offsetof(nc_paged_options, {f}), sizeof(((nc_paged_options *)0)->{f}));')
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["return 0; }"]) + "\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o",
                    str(exe)], check=True)
    seen = dict((a, (int(b), int(c))) for a, b, c in
                (x.split() for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()))
    assert seen["-"] == (ctypes.sizeof(nc.PagedOptions), ctypes.alignment(nc.PagedOptions))
    for f, t in nc.PagedOptions._fields_:
        assert seen[f] == (getattr(nc.PagedOptions, f).offset, ctypes.sizeof(t)), f


def test_buffer_blocks_match_binding(tmp_path):
    """The binding packs a call's pointers and lengths as 8-byte words in the structs' order."""
    fields = {"build": "cached_lens cached_len new_lens new_len free_pages free_len cursor cursor_len block_table "
                       "table_len seq_lens seq_len row_offsets offsets_len slots slots_len counts counts_len",
              "append": "k_rows k_rows_len v_rows v_rows_len slots slots_len k_cache k_len v_cache v_len num_rows",
              "decode": "q q_len k_cache k_len v_cache v_len block_table table_len seq_lens lens_len o o_len workspace "
                        "workspace_bytes"}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "notcute_paged.h"', "int main(void) {"]
    for name, fs in fields.items():
        lines.append(f'printf("%zu", sizeof(nc_paged_{name}_buffers));')
        lines += [f'printf(" %zu", offsetof(nc_paged_{name}_buffers, {f}));' for f in fs.split()]
        lines.append('printf("\\n");')
    src = tmp_path / "blocks.c"
    src.write_text("\n".join(lines + ["return 0; }"]) + "\n")
    exe = tmp_path / "blocks"
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()
    packs = (nc._BUILD_BUFFERS, nc._APPEND_BUFFERS, nc._DECODE_BUFFERS)
    for line, fs, pack in zip(out, fields.values(), packs):
        n = len(fs.split())
        assert [int(x) for x in line.split()] == [8 * n] + [8 * i for i in range(n)]
        assert pack.size == 8 * n


def test_null_blocks_are_refused():
    for name in ("build", "append", "decode"):
        f = getattr(nc.lib(), f"nc_paged_{name}")
        assert nc.STATUS_NAMES[f(0x10, None, ctypes.byref(good()), None)] == INVALID
        assert nc.STATUS_NAMES[f(0x10, bytes(144), None, None)] == INVALID


def test_defaults():
    o = nc.PagedOptions()
    nc.lib().nc_paged_options_init(ctypes.byref(o))
    assert {f: getattr(o, f) for f, _ in o._fields_ if getattr(o, f)} == {
        "num_seqs": 1, "num_q_heads": 1, "num_kv_heads": 1, "max_pages": 1}
    nc.paged_validate(good())
    assert nc.paged_options(head_dim=16, page_size=1, num_pages=1).scale == 0.25


@pytest.mark.parametrize("kw,want", [
    (dict(num_seqs=0), INVALID), (dict(num_q_heads=0), INVALID), (dict(num_kv_heads=0), INVALID),
    (dict(page_size=0), INVALID), (dict(num_pages=0), INVALID), (dict(max_pages=0), INVALID),
    (dict(head_dim=0), INVALID), (dict(head_dim=48), INVALID), (dict(head_dim=256), INVALID),
    (dict(num_q_heads=7), INVALID), (dict(num_q_heads=1), INVALID),
    (dict(table_stride=9), INVALID),
    (dict(token_stride=56), INVALID),                      # rows overlap
    (dict(token_stride=68), INVALID),                      # no multiple of 16 bytes
    (dict(token_stride=64, head_stride=64 * 15), INVALID), # heads overlap
    (dict(token_stride=128, head_stride=64, page_stride=16 * 128 - 64), INVALID),
    (dict(q_head_stride=32), INVALID), (dict(o_stride=8 * 64 - 1), INVALID), (dict(o_head_stride=63), INVALID),
    (dict(row_head_stride=32), INVALID), (dict(row_stride=64), INVALID),
    (dict(num_pages=2 ** 27), OVERFLOW), (dict(max_pages=2 ** 27), OVERFLOW), (dict(num_seqs=2 ** 31), OVERFLOW),
    (dict(num_seqs=2 ** 20, max_pages=2 ** 20), OVERFLOW), (dict(page_stride=2 ** 61), OVERFLOW),
    (dict(page_stride=2 ** 58), OVERFLOW), (dict(token_stride=2 ** 58), OVERFLOW), (dict(o_stride=2 ** 60), OVERFLOW),
    (dict(q_head_stride=2 ** 59), OVERFLOW), (dict(row_head_stride=2 ** 60), OVERFLOW),
    (dict(num_seqs=-1), OVERFLOW),
])
def test_validate_refuses(kw, want):
    with pytest.raises(nc.NcError) as e:
        nc.paged_validate(good(**kw))
    assert e.value.name == want
    assert nc.paged_workspace_bytes(good(**kw)) == 0


@pytest.mark.parametrize("kw", [
    dict(), dict(page_size=1, num_pages=2 ** 31 - 1), dict(page_size=7), dict(num_q_heads=2), dict(num_q_heads=46),
    dict(token_stride=128, head_stride=64), dict(token_stride=72), dict(table_stride=11),
    dict(token_stride=2 * 2 * 64, head_stride=2 * 64, page_stride=16 * 256),  # K and V interleaved
    dict(row_stride=12 * 64), dict(row_stride=131), dict(q_stride=513, o_stride=515),
])
def test_validate_accepts(kw):
    nc.paged_validate(good(**kw))
    assert nc.paged_workspace_bytes(good(**kw)) > 0


def test_validate_counts_a_requests_outputs():
    """num_q_heads * head_dim is an index of 32 bits in the kernels: 2^31 of them are refused, one head less is not."""
    most = dict(num_kv_heads=1, head_dim=64, num_seqs=1, page_size=16, num_pages=4, max_pages=4)
    nc.paged_validate(nc.paged_options(num_q_heads=2 ** 25 - 1, **most))
    with pytest.raises(nc.NcError) as e:
        nc.paged_validate(nc.paged_options(num_q_heads=2 ** 25, **most))
    assert e.value.name == OVERFLOW


def test_unknown_element_type():
    o = good()
    o.element_type = 2
    with pytest.raises(nc.NcError):
        nc.paged_validate(o)


class Fake:
    """A buffer that is only an address: every refused call must return before it is used."""

    def __init__(self, ptr, count, size):
        self.ptr, self.nbytes = ptr, count * size


class FakeModule:
    handle = 0x10


def build_buffers(o, places=64, free=20):
    at = iter(range(0x10000, 0x1000000, 0x10000))
    n = o.num_seqs
    return dict(cached_lens=Fake(next(at), n, 4), new_lens=Fake(next(at), n, 4), free_pages=Fake(next(at), free, 4),
                cursor=Fake(next(at), 1, 4), block_table=Fake(next(at), n * o.max_pages, 4),
                seq_lens=Fake(next(at), n, 4), row_offsets=Fake(next(at), n + 1, 4), slots=Fake(next(at), places, 4),
                counts=Fake(next(at), 4, 4))


@pytest.mark.parametrize("name", ["cached_lens", "new_lens", "cursor", "block_table", "seq_lens", "row_offsets", "counts"])
def test_build_refuses_short_null_and_misaligned(name):
    o = good()
    for change in (lambda b: Fake(b.ptr, b.nbytes // 4 - 1, 4), lambda b: Fake(0, b.nbytes // 4, 4),
                   lambda b: Fake(b.ptr + 2, b.nbytes // 4, 4)):
        bufs = build_buffers(o)
        bufs[name] = change(bufs[name])
        with pytest.raises(nc.NcError) as e:
            nc.paged_build(FakeModule, opts=o, **bufs)
        assert e.value.name == INVALID


@pytest.mark.parametrize("name", ["free_pages", "slots"])
def test_build_refuses_null_of_a_length(name):
    o = good()
    bufs = build_buffers(o)
    bufs[name] = Fake(0, 5, 4)
    with pytest.raises(nc.NcError) as e:
        nc.paged_build(FakeModule, opts=o, **bufs)
    assert e.value.name == INVALID


OUT = ["seq_lens", "counts", "block_table", "row_offsets", "slots"]


@pytest.mark.parametrize("out", OUT)
@pytest.mark.parametrize("other", OUT + ["cached_lens", "cursor", "new_lens", "free_pages"])
def test_build_refuses_overlap(out, other):
    if out == other:
        return
    o = good()
    bufs = build_buffers(o)
    # the output's last element is the other buffer's first (so not the permitted aliasing either)
    bufs[out] = Fake(bufs[other].ptr - bufs[out].nbytes + 4, bufs[out].nbytes // 4, 4)
    with pytest.raises(nc.NcError) as e:
        nc.paged_build(FakeModule, opts=o, **bufs)
    assert e.value.name == INVALID


def append_buffers(o, rows=5):
    cache = o.num_pages * o.num_kv_heads * o.page_size * o.head_dim
    return dict(k_rows=Fake(0x100000, rows * o.num_kv_heads * o.head_dim, 2),
                v_rows=Fake(0x200000, rows * o.num_kv_heads * o.head_dim, 2), slots=Fake(0x300000, rows, 4),
                k_cache=Fake(0x400000, cache, 2), v_cache=Fake(0x800000, cache, 2))


@pytest.mark.parametrize("name", ["k_rows", "v_rows", "slots", "k_cache", "v_cache"])
def test_append_refuses_short_and_null(name):
    o = good()
    for change in (lambda b: Fake(b.ptr, b.nbytes // 2 - 1, 2), lambda b: Fake(0, b.nbytes // 2, 2)):
        bufs = append_buffers(o)
        bufs[name] = change(bufs[name])
        with pytest.raises(nc.NcError) as e:
            nc.paged_append(FakeModule, opts=o, num_rows=5, **bufs)
        assert e.value.name == INVALID


def test_append_refuses_misaligned_overlapping_and_negative():
    o = good()
    for name, by in (("k_cache", 2), ("v_cache", 8), ("slots", 2), ("k_rows", 1)):
        bufs = append_buffers(o)
        bufs[name].ptr += by
        with pytest.raises(nc.NcError):
            nc.paged_append(FakeModule, opts=o, **bufs)
    bufs = append_buffers(o)
    bufs["v_cache"].ptr = bufs["k_cache"].ptr
    with pytest.raises(nc.NcError):
        nc.paged_append(FakeModule, opts=o, **bufs)
    for name in ("k_rows", "slots"):
        bufs = append_buffers(o)
        bufs[name].ptr = bufs["v_cache"].ptr + 64
        with pytest.raises(nc.NcError):
            nc.paged_append(FakeModule, opts=o, **bufs)
    with pytest.raises(ValueError):
        nc.paged_append(FakeModule, opts=o, num_rows=-1, **append_buffers(o))
    # more rows than slots, than the rows' buffer, than 32 bits
    for n, want in ((6, INVALID), (2 ** 31, OVERFLOW)):
        with pytest.raises(nc.NcError) as e:
            nc.paged_append(FakeModule, opts=o, num_rows=n, **append_buffers(o))
        assert e.value.name == want
    nc.paged_append(FakeModule, opts=o, num_rows=0, **append_buffers(o))  # nothing to do, nothing touched


@pytest.mark.parametrize("strides", [
    dict(), dict(token_stride=128), dict(token_stride=2 * 2 * 64, head_stride=2 * 64, page_stride=16 * 256),
    dict(token_stride=128, head_stride=64), dict(token_stride=72, page_stride=4096), dict(num_pages=1, page_stride=8),
    dict(page_size=1, num_pages=9, token_stride=8, head_stride=64), dict(num_kv_heads=1, num_q_heads=1, head_stride=8)])
def test_append_refuses_rows_of_k_and_v_that_meet(strides):
    """V at every 16-byte distance from K: refused exactly where some row of V holds an element of a row of K.
    With no rows to append, an accepted call launches nothing."""
    o = good(**dict(dict(num_pages=3), **strides))
    nc.paged_validate(o)
    d, ps, H, P = o.head_dim, o.page_size, o.num_kv_heads, o.num_pages
    ts = o.token_stride or d
    hs = o.head_stride or ps * ts
    pg = o.page_stride or max(H * hs, ps * ts)
    at = (np.arange(P)[:, None, None] * pg + np.arange(H)[None, :, None] * hs + np.arange(ps)[None, None, :] * ts).ravel()
    held = np.zeros(at.max() + d, dtype=bool)
    held[(at[:, None] + np.arange(d)).ravel()] = True
    n = held.size
    for delta in list(range(8, min(n, 1600), 8)) + [n // 8 * 8 - 8, n // 8 * 8, (n + 7) // 8 * 8]:
        meet = bool(np.any(held[delta:] & held[:n - delta])) if delta < n else False
        for sign in (1, -1):
            bufs = append_buffers(o)
            bufs["k_cache"] = Fake(0x4000000, n, 2)
            bufs["v_cache"] = Fake(0x4000000 + sign * 2 * delta, n, 2)
            try:
                nc.paged_append(FakeModule, opts=o, num_rows=0, **bufs)
                refused = False
            except nc.NcError as e:
                assert e.name == INVALID
                refused = True
            assert refused == meet, (delta, sign)


def decode_buffers(o):
    cache = o.num_pages * o.num_kv_heads * o.page_size * o.head_dim
    qo = o.num_seqs * o.num_q_heads * o.head_dim
    return dict(q=Fake(0x100000, qo, 2), k_cache=Fake(0x200000, cache, 2), v_cache=Fake(0x600000, cache, 2),
                block_table=Fake(0xa00000, o.num_seqs * o.max_pages, 4), seq_lens=Fake(0xb00000, o.num_seqs, 4),
                o=Fake(0xc00000, qo, 4), workspace=Fake(0x10000000, nc.paged_workspace_bytes(o), 1))


@pytest.mark.parametrize("name", ["q", "k_cache", "v_cache", "block_table", "seq_lens", "o", "workspace"])
def test_decode_refuses_short_and_null(name):
    o = good()
    for change in (lambda b: Fake(b.ptr, b.nbytes - 1, 1), lambda b: Fake(0, b.nbytes, 1)):
        bufs = decode_buffers(o)
        bufs[name] = change(bufs[name])
        with pytest.raises(nc.NcError) as e:
            nc.paged_decode(FakeModule, opts=o, **bufs)
        assert e.value.name == INVALID


def test_decode_refuses_misaligned_and_overlapping():
    o = good()
    for name, by in (("q", 1), ("k_cache", 8), ("v_cache", 2), ("block_table", 2), ("seq_lens", 1), ("o", 2),
                     ("workspace", 8)):
        bufs = decode_buffers(o)
        bufs[name].ptr += by
        with pytest.raises(nc.NcError) as e:
            nc.paged_decode(FakeModule, opts=o, **bufs)
        assert e.value.name == INVALID, name
    for out in ("o", "workspace"):
        for other in ("q", "k_cache", "v_cache", "block_table", "seq_lens", "workspace"):
            if out == other:
                continue
            bufs = decode_buffers(o)
            bufs[out].ptr = bufs[other].ptr
            with pytest.raises(nc.NcError) as e:
                nc.paged_decode(FakeModule, opts=o, **bufs)
            assert e.value.name == INVALID, (out, other)


def test_no_module_is_refused():
    class None_:
        handle = None

    o = good()
    for call, bufs in ((nc.paged_build, build_buffers(o)), (nc.paged_append, append_buffers(o)),
                       (nc.paged_decode, decode_buffers(o))):
        with pytest.raises(nc.NcError) as e:
            call(None_, opts=o, **bufs)
        assert e.value.name == INVALID


def test_index_arithmetic(tmp_path):
    """The quotient by a page size for every divisor class and the dividends next to its multiples up to
    2^31 - 1, and the cut of a length, compiled from the header that the kernels include."""
    src = tmp_path / "index.cpp"
    src.write_text(r"""
#include <cstdio>
#include <cstdint>
#include "paged_args.h"
int main() {
    const uint32_t most = 0x7fffffffu;
    uint64_t x = 88172645463325252ull;
    for (uint64_t k = 0; k < 6000; ++k) {
        x ^= x << 13; x ^= x >> 7; x ^= x << 17;
        uint32_t d = k < 3000 ? (uint32_t)k + 1 : (uint32_t)(x % most) + 1;
        if (k % 5 == 0) d = 1u << (k / 5 % 31);
        const nc_paged_div v = nc_paged_make_div(d);
        for (int i = 0; i < 400; ++i) {
            x ^= x << 13; x ^= x >> 7; x ^= x << 17;
            uint32_t n = (uint32_t)(x % ((uint64_t)most + 1));
            if (i % 4 == 1) n = n / d * d;
            if (i % 4 == 2 && n / d) n = n / d * d - 1;
            if (i == 0) n = most;
            if (i == 4) n = most / d * d - (d > 1);
            if (nc_paged_quot(n, v) != n / d) { std::printf("%u / %u\n", n, d); return 1; }
        }
    }
    // shares of nc_paged_each() cover all units with no more workgroups than there are, and no smaller one does
    for (int k = 0; k < 20000; ++k) {
        x ^= x << 13; x ^= x >> 7; x ^= x << 17;
        const uint32_t units = k % 2 ? (uint32_t)(x % 5000) + 1 : (uint32_t)(x % (1u << 30)) + 1;
        const uint32_t lg = (uint32_t)((x >> 32) % 12), n = 1u << lg, least = k % 3 ? 1 : (uint32_t)(x % 17) + 1;
        const uint32_t each = nc_paged_each(units, lg, least);
        if (each < least || (uint64_t)each * n < units || (each > least && (uint64_t)(each - 1) * n >= units)) return 3;
    }
    for (uint32_t g = 1; g < 300; ++g) {  // the waves' and parts' query heads cover the group, 16 a wave
        const uint32_t rows = g < 64 ? g : 64, sh = nc_paged_wave_shift(rows);
        if ((16u << sh) < rows || (sh && (8u << sh) >= rows) || nc_paged_head_parts(g) * 64 < g || (nc_paged_head_parts(g) - 1) * 64 >= g) return 4;
    }
    // the join's rounds and LDS suffice for every size of piece
    for (uint32_t d = 16; d <= 128; d *= 2)
        for (uint32_t rows = 1; rows <= 64; ++rows) {
            const uint32_t fan = nc_paged_fan(rows, d);
            uint64_t most_pieces = 1;
            for (uint32_t i = 0; i < NC_PAGED_ROUNDS; ++i) most_pieces *= fan;
            if (most_pieces < NC_PAGED_MAX_WGS || fan > 16 || fan * rows > NC_PAGED_MERGE_ROWS) return 6;
        }
    if (nc_paged_cut(-1, 5) != 0 || nc_paged_cut(INT32_MIN, 5) != 0 || nc_paged_cut(4, 5) != 4 ||
        nc_paged_cut(INT32_MAX, 5) != 5) return 2;
    return 0;
}
""")
    exe = tmp_path / "index"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Wextra", "-Werror", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout


def test_reference_against_a_direct_softmax():
    """The tests' own reference: one request with an absent page against a softmax over the rest."""
    rng = np.random.default_rng(1)
    pool = pc.Pool(rng, 6, 1, 4, 16)
    table = np.array([[2, 99, 0, -1]], dtype=np.int32)
    q = pc.encode(rng.standard_normal((1, 1, 16)), "f16")
    o, _ = pc.ref_decode(q, pool, table, [10], 0.25, 1)
    rows = [(2, t) for t in range(4)] + [(0, t) for t in range(2)]
    k = np.array([pc.decode_bits(pool.get(0, p, 0, t), "f16") for p, t in rows])
    v = np.array([pc.decode_bits(pool.get(1, p, 0, t), "f16") for p, t in rows])
    p = np.exp(0.25 * (k @ pc.decode_bits(q, "f16")[0, 0]))
    assert np.allclose(o[0, 0], (p / p.sum()) @ v, atol=1e-14)
