"""Paged cache, on the CPU: index arithmetic and counts of csrc/paged_args.h beyond those of test_paged.py."""

import os
import re
import subprocess

import pytest

import notcute_flash as nc

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "not-cute-zig_amd", "csrc")


def run_cpp(tmp_path, body):
    src, exe = tmp_path / "x.cpp", tmp_path / "x"
    src.write_text('#include <cstdio>\n#include <cstdint>\n#include "paged_args.h"\nint main() {\n' + body + "\nreturn 0; }\n")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Wextra", "-Werror", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout


def test_divisor_of_neighbouring_heads(tmp_path):
    """The divisor of heads taken 2 or 4 at a time, made from the heads' own."""
    run_cpp(tmp_path, r"""
    uint64_t x = 88172645463325252ull;
    for (uint32_t k = 1; k < 20000; ++k) {
        for (uint32_t side = 0; side < 3; ++side) {
            const uint32_t d = (k < 5000 ? k : k * 40009u % (1u << 28)) << side;
            if (!d) continue;
            const nc_paged_div v = nc_paged_div_by(nc_paged_make_div(d), side);
            if (v.d != d >> side) return 1;
            for (int i = 0; i < 8; ++i) {
                x ^= x << 13; x ^= x >> 7; x ^= x << 17;
                uint32_t n = (uint32_t)(x & 0x7fffffffu);
                if (i % 2) n = n / v.d * v.d - (i % 4 == 1 && n >= v.d);
                if (i == 0) n = 0x7fffffffu;
                if (nc_paged_quot(n, v) != n / v.d) { std::printf("%u / %u\n", n, v.d); return 2; }
            }
        }
    }""")


@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("group", [1, 16, 17, 32, 33, 64, 65, 128, 129, 1000])
@pytest.mark.parametrize("heads", [1, 3])
def test_blocks_that_the_header_promises_to_accept(d, group, heads):
    """The header's count of blocks: as many as it names are accepted, and 8 times as many (32-token blocks, of which a wave's
    step may hold up to 8) are not."""
    text = " ".join(re.sub(r"\n \*", " ", open(os.path.join(ROOT, "include", "notcute_paged.h")).read()).split())
    assert "for each request, key head and part of up to 64 of the key head's query heads, a block for every 32 tokens of the table's row and two more" in text
    parts, tokens = -(-group // 64), 2 ** 20
    seqs = 2 ** 30 // (heads * parts * (tokens // 32 + 2))
    o = dict(num_q_heads=heads * group, num_kv_heads=heads, head_dim=d, page_size=16, num_pages=4, max_pages=tokens // 16)
    nc.paged_validate(nc.paged_options(num_seqs=seqs, **o))
    with pytest.raises(nc.NcError) as e:
        nc.paged_validate(nc.paged_options(num_seqs=8 * seqs + 8, **o))
    assert e.value.name == "Overflow"
