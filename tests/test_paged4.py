"""The smaller paged cache, on the CPU: the C ABI of include/notcute_paged4.h, its refusals, and the definitions that the GPU tests
compare with."""

import ctypes
import os
import re
import subprocess

import numpy as np
import pytest

import notcute_flash as nc
import paged4check as p4

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "notcute_paged4.h")
INVALID, OVERFLOW = "InvalidValue", "Overflow"


class FakeBuffer:
    """An address and a size that nothing reads: for calls that are refused."""

    def __init__(self, ptr, nbytes):
        self.ptr, self.nbytes = ptr, nbytes


class FakeModule:
    handle = 0x10


def good(**kw):
    base = dict(num_seqs=4, num_q_heads=8, num_kv_heads=2, head_dim=64, page_size=16, num_pages=50, max_pages=10)
    base.update(kw)
    return nc.paged_options(**base)


def test_library_exports_every_declared_function():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(nc_paged[a-z0-9_]+)\s*\(", text)))
    assert len(names) == 10
    for n in names:
        assert hasattr(nc.load_library(), n), n
        assert n in nc._SIGS, n


def test_blocks_match_binding(tmp_path):
    """The binding packs a call's pointers and lengths as 8-byte words in the structs' order."""
    cache = "cache.k cache.k_len cache.v cache.v_len cache.k_scales cache.k_scales_len cache.v_scales cache.v_scales_len"
    lists = ("block_table table_len seq_lens lens_len mass.mass mass.mass_len mass.mass_stride free_pages free_len cursor cursor_len "
             "kept_lens kept_len counts counts_len workspace workspace_bytes")
    lists = " ".join("lists." + x for x in lists.split())
    blocks = [("nc_paged4_append_buffers", "k_rows k_rows_len v_rows v_rows_len slots slots_len " + cache + " num_rows", nc._ROWS4_BUFFERS),
              ("nc_paged4_read_buffers", cache + " slots slots_len k_rows k_rows_len v_rows v_rows_len num_rows", nc._ROWS4_BUFFERS),
              ("nc_paged4_decode_buffers", "q q_len " + cache + " block_table table_len seq_lens lens_len o o_len workspace workspace_bytes",
               nc._DECODE4_BUFFERS),
              ("nc_paged_mass", "mass mass_len mass_stride", nc._MASS),
              ("nc_paged_evict_buffers", lists + " k_cache k_len v_cache v_len", nc._EVICT_BUFFERS),
              ("nc_paged4_evict_buffers", lists + " " + cache, nc._EVICT4_BUFFERS),
              ("nc_paged_evict_rules", "limit budget sinks recent", None)]
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "notcute_paged4.h"', "int main(void) {"]
    for name, fs, _ in blocks:
        lines.append(f'printf("%zu", sizeof({name}));')
        lines += [f'printf(" %zu", offsetof({name}, {f}));' for f in fs.split()]
        lines.append('printf("\\n");')
    src, exe = tmp_path / "blocks.c", tmp_path / "blocks"
    src.write_text("\n".join(lines + ["return 0; }"]) + "\n")
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()
    for line, (_, fs, pack) in zip(out, blocks):
        n = len(fs.split())
        assert [int(x) for x in line.split()] == [8 * n] + [8 * i for i in range(n)]
        assert pack is None or pack.size == 8 * n
    assert ctypes.sizeof(nc.EvictRules) == 32 and [f for f, _ in nc.EvictRules._fields_] == ["limit", "budget", "sinks", "recent"]


@pytest.mark.parametrize("kw,want", [
    (dict(head_dim=16), INVALID), (dict(head_dim=48), INVALID), (dict(token_stride=72), INVALID), (dict(token_stride=80), INVALID),
    (dict(token_stride=96, head_stride=64), INVALID), (dict(page_stride=2 * 16 * 64 + 16), INVALID), (dict(num_q_heads=7), INVALID),
    (dict(max_pages=2 ** 27), OVERFLOW), (dict(num_pages=2 ** 26 + 1, page_stride=2048), OVERFLOW),
    (dict(num_pages=2 ** 26), OVERFLOW),
])
def test_validate_refuses(kw, want):
    with pytest.raises(nc.NcError) as e:
        nc.paged4_validate(good(**kw))
    assert e.value.name == want
    assert nc.paged4_workspace_bytes(good(**kw)) == 0 and nc.paged4_workspace_bytes(good(**kw), mass=True) == 0


@pytest.mark.parametrize("kw", [dict(), dict(head_dim=32), dict(head_dim=128), dict(token_stride=96), dict(page_size=7),
                                dict(token_stride=128, head_stride=64), dict(num_q_heads=200), dict(dtype="bf16"), dict(num_pages=2 ** 26 - 1)])
def test_validate_accepts_and_workspaces_grow(kw):
    nc.paged4_validate(good(**kw))
    o = good(**kw)
    plain, mass = nc.paged4_workspace_bytes(o), nc.paged4_workspace_bytes(o, mass=True)
    room = -(-o.max_pages * o.page_size // 16) * 16
    assert plain > 0 and mass > 4 * o.num_seqs * o.num_q_heads * room
    assert nc.paged_mass_workspace_bytes(o) > 4 * o.num_seqs * o.num_q_heads * room
    assert nc.paged_evict_workspace_bytes(o) >= 8 * o.num_seqs * o.max_pages * o.page_size


def cache_bytes(o):
    n = o.num_pages * o.num_kv_heads * o.page_size * o.head_dim
    return n // 2, n // 32


def rows_call(o, which="append", **kw):
    c, s = cache_bytes(o)
    rows = 5
    b = dict(k_rows=FakeBuffer(0x100000, rows * 128 * 2), v_rows=FakeBuffer(0x200000, rows * 128 * 2), slots=FakeBuffer(0x300000, rows * 4),
             k=FakeBuffer(0x1000000, c), v=FakeBuffer(0x2000000, c), ks=FakeBuffer(0x3000000, s), vs=FakeBuffer(0x4000000, s))
    b.update(kw)
    if which == "append":
        nc.paged4_append(FakeModule(), b["k_rows"], b["v_rows"], b["slots"], b["k"], b["v"], b["ks"], b["vs"], o)
    else:
        nc.paged4_read(FakeModule(), b["k"], b["v"], b["ks"], b["vs"], b["slots"], b["k_rows"], b["v_rows"], o)


@pytest.mark.parametrize("which", ["append", "read"])
@pytest.mark.parametrize("kw", [
    dict(k=FakeBuffer(0, 1 << 20)), dict(ks=FakeBuffer(0, 1 << 20)), dict(v=FakeBuffer(0x2000008, 1 << 20)),
    dict(k=FakeBuffer(0x1000000, 51199)), dict(vs=FakeBuffer(0x4000000, 3199)), dict(k_rows=FakeBuffer(0x100001, 1 << 20)),
    dict(v_rows=FakeBuffer(0x200000, 5 * 128 * 2 - 2)), dict(slots=FakeBuffer(0x300002, 20)), dict(slots=FakeBuffer(0, 20)),
    dict(k_rows=FakeBuffer(0x1000000, 1 << 20)), dict(v_rows=FakeBuffer(0x4000000 - 100, 1 << 20)),
])
def test_rows_calls_refuse(which, kw):
    with pytest.raises(nc.NcError) as e:
        rows_call(good(), which, **kw)
    assert e.value.name == INVALID


def test_append_refuses_parts_that_share_memory():
    o = good()
    c, s = cache_bytes(o)
    for kw in (dict(v=FakeBuffer(0x1000000, c)), dict(vs=FakeBuffer(0x3000000 + s - 1, s)), dict(ks=FakeBuffer(0x1000000 + c - 1, s)),
               dict(slots=FakeBuffer(0x3000000, 20))):
        with pytest.raises(nc.NcError) as e:
            rows_call(o, "append", **kw)
        assert e.value.name == INVALID


def test_read_refuses_outputs_that_share_memory():
    for kw in (dict(v_rows=FakeBuffer(0x100000 + 64, 1 << 20)), dict(slots=FakeBuffer(0x100000, 20)), dict(slots=FakeBuffer(0x200400, 20))):
        with pytest.raises(nc.NcError) as e:
            rows_call(good(), "read", **kw)
        assert e.value.name == INVALID


def test_rows_of_zero_do_nothing_but_a_bad_cache_is_refused():
    o = good()
    c, s = cache_bytes(o)
    b = [FakeBuffer(0x1000000, c), FakeBuffer(0x2000000, c), FakeBuffer(0x3000000, s), FakeBuffer(0x4000000, s)]
    none = FakeBuffer(0, 0)
    nc.paged4_append(FakeModule(), none, none, none, *b, o)
    nc.paged4_read(FakeModule(), *b, none, none, none, o)
    for call in (lambda: nc.paged4_append(FakeModule(), none, none, none, b[0], b[1], b[2], none, o),
                 lambda: nc.paged4_read(FakeModule(), b[0], none, b[2], b[3], none, none, none, o)):
        with pytest.raises(nc.NcError):
            call()
    with pytest.raises(ValueError):
        nc.paged4_append(FakeModule(), none, none, none, *b, o, num_rows=-1)


def decode_call(o, four, **kw):
    c, s = cache_bytes(o)
    mass_ws = nc.paged4_workspace_bytes(o, mass=True) if four else nc.paged_mass_workspace_bytes(o)
    b = dict(q=FakeBuffer(0x100000, 4 * 8 * 64 * 2), k=FakeBuffer(0x1000000, 4 * c), v=FakeBuffer(0x2000000, 4 * c), ks=FakeBuffer(0x3000000, s),
             vs=FakeBuffer(0x4000000, s), table=FakeBuffer(0x200000, 160), lens=FakeBuffer(0x300000, 16), out=FakeBuffer(0x400000, 4 * 8 * 64 * 4),
             mass=FakeBuffer(0x500000, 4 * 160 * 4), work=FakeBuffer(0x6000000, mass_ws), mass_stride=0)
    b.update(kw)
    if four:
        nc.paged4_decode(FakeModule(), b["q"], b["k"], b["v"], b["ks"], b["vs"], b["table"], b["lens"], b["out"], b["work"], o, mass=b["mass"],
                         mass_stride=b["mass_stride"])
    else:
        nc.paged_decode_mass(FakeModule(), b["q"], b["k"], b["v"], b["table"], b["lens"], b["out"], b["mass"], b["work"], o,
                             mass_stride=b["mass_stride"])


@pytest.mark.parametrize("four", [True, False])
@pytest.mark.parametrize("kw", [
    dict(q=FakeBuffer(0, 4096)), dict(k=FakeBuffer(0x1000001, 1 << 22)), dict(table=FakeBuffer(0x200000, 159)), dict(lens=FakeBuffer(0x300000, 12)),
    dict(out=FakeBuffer(0x400002, 1 << 16)), dict(out=FakeBuffer(0x400000, 4 * 8 * 64 * 4 - 4)), dict(work=FakeBuffer(0x6000008, 1 << 30)),
    dict(mass=FakeBuffer(0, 1 << 16)), dict(mass=FakeBuffer(0x500000, 4 * 160 * 4 - 4)), dict(mass=FakeBuffer(0x500002, 1 << 16)),
    dict(mass_stride=159), dict(mass=FakeBuffer(0x400000, 1 << 16)), dict(mass=FakeBuffer(0x300000, 1 << 16)), dict(mass=FakeBuffer(0x6000000, 1 << 16)),
    dict(mass=FakeBuffer(0x100000, 1 << 16)), dict(mass=FakeBuffer(0x1000100, 1 << 16)), dict(out=FakeBuffer(0x1000000, 1 << 16)),
])
def test_decodes_with_a_mass_refuse(four, kw):
    with pytest.raises(nc.NcError) as e:
        decode_call(good(), four, **kw)
    assert e.value.name == INVALID


def test_decodes_refuse_a_workspace_without_room_for_scores():
    o = good()
    for four, small in ((True, nc.paged4_workspace_bytes(o)), (False, nc.paged_workspace_bytes(o))):
        with pytest.raises(nc.NcError) as e:
            decode_call(o, four, work=FakeBuffer(0x6000000, small))
        assert e.value.name == INVALID


def test_decode_refuses_scales_that_o_overlaps():
    with pytest.raises(nc.NcError) as e:
        decode_call(good(), True, out=FakeBuffer(0x3000000 - 64, 1 << 16))
    assert e.value.name == INVALID


def evict_call(o, four, rules=None, **kw):
    c, s = cache_bytes(o)
    b = dict(table=FakeBuffer(0x200000, 160), lens=FakeBuffer(0x300000, 16), mass=FakeBuffer(0x500000, 4 * 160 * 4), free=FakeBuffer(0x600000, 200),
             cursor=FakeBuffer(0x700000, 4), kept=FakeBuffer(0x800000, 16), counts=FakeBuffer(0x900000, 16),
             work=FakeBuffer(0x6000000, nc.paged_evict_workspace_bytes(o)), k=FakeBuffer(0x1000000, 4 * c), v=FakeBuffer(0x2000000, 4 * c),
             ks=FakeBuffer(0x3000000, s), vs=FakeBuffer(0x4000000, s), mass_stride=0)
    b.update(kw)
    rules = rules or nc.evict_rules(limit=64, budget=32, sinks=4, recent=8)
    cache = [b["k"], b["v"]] + ([b["ks"], b["vs"]] if four else [])
    f = nc.paged4_evict if four else nc.paged_evict
    f(FakeModule(), b["table"], b["lens"], b["mass"], *cache, b["free"], b["cursor"], b["kept"], b["counts"], b["work"], rules, o,
      mass_stride=b["mass_stride"])


@pytest.mark.parametrize("four", [True, False])
@pytest.mark.parametrize("kw", [
    dict(table=FakeBuffer(0x200000, 156)), dict(lens=FakeBuffer(0, 16)), dict(mass=FakeBuffer(0x500000, 100)), dict(mass_stride=100),
    dict(free=FakeBuffer(0, 200)), dict(free=FakeBuffer(0x600001, 200)), dict(cursor=FakeBuffer(0, 4)), dict(kept=FakeBuffer(0x800000, 12)),
    dict(counts=FakeBuffer(0x900000, 12)), dict(work=FakeBuffer(0x6000000, 100)), dict(work=FakeBuffer(0x6000008, 1 << 20)),
    dict(k=FakeBuffer(0x1000000, 100)), dict(v=FakeBuffer(0x1000000, 1 << 20)), dict(kept=FakeBuffer(0x300004, 16)),
    dict(counts=FakeBuffer(0x6FFFFC, 16)), dict(free=FakeBuffer(0x200000, 200)), dict(mass=FakeBuffer(0x1000000, 1 << 16)),
    dict(free=FakeBuffer(0x2000000, 200)), dict(kept=FakeBuffer(0x900000, 16)), dict(lens=FakeBuffer(0x500000, 16)),
    dict(rules=nc.evict_rules(limit=31, budget=32)), dict(rules=nc.evict_rules(limit=64, budget=0)),
    dict(rules=nc.evict_rules(limit=64, budget=32, sinks=33)), dict(rules=nc.evict_rules(limit=64, budget=32, sinks=30, recent=3)),
    dict(rules=nc.evict_rules(limit=64, budget=32, sinks=2 ** 64 - 1, recent=2)),
])
def test_evictions_refuse(four, kw):
    with pytest.raises(nc.NcError) as e:
        evict_call(good(), four, **kw)
    assert e.value.name == INVALID


def test_evictions_refuse_too_many_requests():
    o = nc.paged_options(num_seqs=2 ** 20 + 1, num_q_heads=1, head_dim=64, page_size=16, num_pages=50, max_pages=1)
    big = FakeBuffer(0x10000000000, 1 << 40)
    with pytest.raises(nc.NcError) as e:
        evict_call(o, False, table=big, lens=big, mass=big, kept=big, work=big)
    assert e.value.name == OVERFLOW


def test_negative_rules_are_refused():
    for kw in (dict(limit=-1, budget=1), dict(limit=2, budget=-1), dict(limit=2, budget=1, sinks=-1), dict(limit=2, budget=1, recent=-1)):
        with pytest.raises(ValueError):
            nc.evict_rules(**kw)


def test_null_blocks_are_refused():
    lib, o, rules = nc.lib(), ctypes.byref(good()), ctypes.byref(nc.evict_rules(limit=2, budget=1))
    for f in (lib.nc_paged4_append, lib.nc_paged4_read):
        assert nc.STATUS_NAMES[f(0x10, None, o, None)] == INVALID
        assert nc.STATUS_NAMES[f(0x10, bytes(200), None, None)] == INVALID
    for f in (lib.nc_paged4_decode, lib.nc_paged_decode_mass):
        assert nc.STATUS_NAMES[f(0x10, None, bytes(24), o, None)] == INVALID
    assert nc.STATUS_NAMES[lib.nc_paged_decode_mass(0x10, bytes(200), None, o, None)] == INVALID
    for f in (lib.nc_paged_evict, lib.nc_paged4_evict):
        assert nc.STATUS_NAMES[f(0x10, None, rules, o, None)] == INVALID
        assert nc.STATUS_NAMES[f(0x10, bytes(256), rules, o, None)] == INVALID


def test_quantisation_by_the_header():
    """The tests' own definition: scales and codes of values that were worked out by hand, and the bound of half a step."""
    x = np.zeros((4, 32))
    x[0, :4] = 7.0, 5.0, 0.25, -0.75   # k = 0: 7 is 6, ties to the even code
    x[1, 0], x[1, 1] = np.nextafter(7.0, 8), 3.0  # k = 1
    x[2, 5] = -2.0 ** -20
    c, s = p4.quantise(x, "f16")
    assert s[:, 0].tolist() == [127, 128, 105, 104]
    assert c[0, :4].tolist() == [7, 6, 0, 10] and c[1, :2].tolist() == [6, 3] and c[2, 5] == 8 + 6
    assert p4.quantise(np.full((1, 32), 65504.0), "f16")[1][0, 0] == 140
    assert p4.quantise(np.full((1, 32), 3.3e38), "bf16")[1][0, 0] == 252
    x[3, 7] = np.nan
    c, s = p4.quantise(x, "bf16")
    assert s[3, 0] == 255 and not c[3].any() and s[2, 0] == 127 - 22
    rng = np.random.default_rng(0)
    y = rng.standard_normal((500, 32)) * 2.0 ** rng.integers(-10, 10, (500, 1))
    c, s = p4.quantise(y, "f16")
    assert (np.abs(p4.values(c, s) - y) <= 2.0 ** (s.astype(float) - 127) * np.where(np.abs(y) > 4 * 2.0 ** (s.astype(float) - 127), 1.0, 0.5)).all()


def test_eviction_by_the_header():
    lens = np.array([5, 3, 9], np.int32)
    mass = np.array([[5, 1, 1, 2, 0, 9, 9, 9, 9], [1] * 9, [0, 3, 3, 3, np.nan, -0.0, 0.0, 1, 1]], np.float32)
    table = np.array([[4, 7, 2, -1, -1], [1, 3, -1, -1, -1], [0, 9, 8, 6, 5]], np.int32)
    free = np.arange(100, 110, dtype=np.int32)
    kept, out, m, f, counts = p4.ref_evict(lens, mass, table, free, 10, 2, 10, (4, 3, 1, 1))
    assert kept == [[0, 3, 4], None, [0, 4, 8]] and out.tolist() == [3, 3, 3]
    assert m[0].tolist() == [5, 2, 0, 0, 0, 9, 9, 9, 9] and f[:6].tolist() == list(range(100, 106))
    assert f[6:].tolist() == [2, 8, 6, 5] and counts.tolist() == [6, 2, 4, 8]
