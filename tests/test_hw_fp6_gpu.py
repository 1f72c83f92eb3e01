"""The gfx950 instructions that split a query for the 4-bit cache's attention, pinned on the GPU with one-wave probes
(not-cute-zig_amd/csrc/hw_probe.hip): the product of 4-bit rows and 6-bit columns, and the scaled conversions to 6 and 8 bits."""

import ctypes
import os

import numpy as np
import pytest

import notcute_flash as nc

pytestmark = pytest.mark.gpu

PROBE = os.path.join(os.path.dirname(__file__), "..", "not-cute-zig_amd", "hw_probe_gfx950.hsaco")
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6])
E2M3 = np.array([(-1.0) ** (b >> 5) * ((b & 7) / 8 if (b >> 3) & 3 == 0 else (1 + (b & 7) / 8) * 2.0 ** ((b >> 3 & 3) - 1)) for b in range(64)])
E4M3 = np.array([(-1.0) ** (b >> 7) * ((b & 7) / 8 * 2.0 ** -6 if (b >> 3) & 15 == 0 else (1 + (b & 7) / 8) * 2.0 ** ((b >> 3 & 15) - 7))
                 for b in range(256)])


@pytest.fixture(scope="module")
def probe(gpu):
    if not os.path.exists(PROBE):
        pytest.fail(f"{PROBE} is missing: run __graft_entry__.build()")
    return nc.Module.load_file(PROBE)


def run(probe, name, ins, outs, *more):
    bufs = [nc.DeviceBuffer.from_array(x) for x in ins] + [nc.DeviceBuffer(4 * n) for n, _ in outs]
    probe.get_function(name).launch((1,), (64,), [ctypes.c_void_p(b.ptr) for b in bufs] + list(more))
    nc.synchronize()
    got = [b.download(t, n) for b, (n, t) in zip(bufs[len(ins):], outs)]
    for b in bufs:
        b.free()
    return got


def pack6(codes):
    """Codes [..., 32] as 6 words each."""
    out = []
    for row in codes.reshape(-1, 32):
        z = sum(int(v) << (6 * j) for j, v in enumerate(row))
        out += [z >> (32 * j) & 0xFFFFFFFF for j in range(6)]
    return np.array(out, np.uint32)


def nearest(values, x):
    """Codes of the nearest of ascending `values`, of two as near the even one, the last above it."""
    d = np.abs(values[None, :] - np.minimum(np.abs(x), values[-1])[:, None])
    near = d == d.min(1, keepdims=True)
    first, last = near.argmax(1), len(values) - 1 - near[:, ::-1].argmax(1)
    return np.where((first != last) & (first % 2 == 1), last, first)


@pytest.mark.parametrize("spread", [0, 8, 24])
@pytest.mark.parametrize("most", [16, 24, 32])  # codes of values below 2, 4, 8
def test_products_of_4_and_6_bits_are_exact(probe, spread, most):
    """Of g = l/16, lane l holds values 32g..+31 of row l%16 and of column l%16, and the scales of both; no product loses a bit, so that
    only the sums' roundings are left (8, as for 8-bit values of at most 2)."""
    rng = np.random.default_rng(spread + most)
    a, b = rng.integers(0, 16, (16, 128)).astype(np.uint8), rng.integers(0, most, (16, 128)) | rng.integers(0, 2, (16, 128)) << 5
    sa, sb = (rng.integers(127 - spread, 128, (16, 4)).astype(np.uint8) for _ in range(2))
    x = E2M1[a] * np.repeat(2.0 ** (sa.astype(float) - 127), 32, axis=1)
    y = E2M3[b] * np.repeat(2.0 ** (sb.astype(float) - 127), 32, axis=1)
    got, = run(probe, "nc_probe_mfma_fp4_fp6", [(a[:, 0::2] | a[:, 1::2] << 4).astype(np.uint8).ravel(), sa.ravel(), pack6(b), sb.ravel()],
               [(256, np.float32)])
    out = np.zeros((16, 16))
    for lane in range(64):
        out[4 * (lane // 16):4 * (lane // 16) + 4, lane % 16] = got[4 * lane:4 * lane + 4]
    if spread == 0:
        assert (out == x @ y.T).all()
    assert np.max(np.abs(out - x @ y.T) / (np.abs(x) @ np.abs(y).T)) <= 8 * 2.0 ** -24


@pytest.mark.parametrize("ka,kb", [(254, 1), (200, 1), (127, 1), (252, 3), (255, 3), (3, 255)])
def test_far_scales_of_4_and_6_bits_cancel(probe, ka, kb):
    a, b = np.full((16, 64), 0x22, np.uint8), pack6(np.full((16, 128), 8))  # all ones
    got, = run(probe, "nc_probe_mfma_fp4_fp6", [a.ravel(), np.full(64, ka, np.uint8), b, np.full(64, kb, np.uint8)], [(256, np.float32)])
    if 255 in (ka, kb):
        assert np.isnan(got).all()
    else:
        assert (got.astype(float) == 128 * 2.0 ** (ka + kb - 254)).all()


def inputs(values, power):
    """Every value, the borders between two and their neighbours, ones above the largest, both zeros; of both signs, times 2^power."""
    mid = (values[1:] + values[:-1]) / 2
    f = mid.astype(np.float32)
    x = np.concatenate([values, mid, np.nextafter(f, np.float32(0)), np.nextafter(f, np.float32(1e9)), [2 * values[-1], 0.0, 2.0 ** -30]])
    x = np.concatenate([x, -x, np.zeros(-2 * len(x) % 32)])
    with np.errstate(over="ignore"):
        y = (x * 2.0 ** power).astype(np.float32)
    keep = np.isfinite(y) & (y.astype(float) == x * 2.0 ** power)  # what f32 holds
    return np.where(keep, y, np.float32(0)), np.where(keep, x, 0.0)


@pytest.mark.parametrize("power", [0, 13, -20, -100, -126, 100])
def test_f32_to_fp6_rounds_to_nearest_even(probe, power):
    y, x = inputs(E2M3[:32], power)
    n = len(y) // 32
    s = np.full(n, 2.0 ** power, np.float32)
    codes, back = run(probe, "nc_probe_fp6_convert", [y, s], [(6 * n, np.uint32), (32 * n, np.float32)], ctypes.c_uint32(n))
    want = nearest(E2M3[:32], x) | np.where(np.signbit(x), 32, 0)
    assert np.array_equal(codes, pack6(want.reshape(n, 32)))
    assert np.array_equal(back.astype(float), E2M3[want] * 2.0 ** power)


@pytest.mark.parametrize("power", [0, 13, -20, -100, -110, 100])
def test_f32_to_scaled_fp8_rounds_to_nearest_even(probe, power):
    """Values of at most 2 scales, as a query's parts are, and less than the least step."""
    values = E4M3[:65]
    y, x = inputs(values, power)
    keep = np.abs(x) <= 2
    y, x = np.where(keep, y, np.float32(0)), np.where(keep, x, 0.0)
    n = len(y) // 4
    s = np.full(n, 2.0 ** power, np.float32)
    codes, back = run(probe, "nc_probe_fp8_scaled", [y, s], [(n, np.uint32), (4 * n, np.float32)], ctypes.c_uint32(n))
    want = nearest(values, x) | np.where(np.signbit(x), 128, 0)
    assert np.array_equal(codes.view(np.uint8), want.astype(np.uint8))
    assert np.array_equal(back.astype(float), E4M3[want] * 2.0 ** power)
