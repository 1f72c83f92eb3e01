"""Shared helpers of the smaller paged cache's tests: 4-bit pools in any layout, the quantisation's definition, references in
float64 and Python integers, and error bounds.

Bound of one output element over a 4-bit cache, beside pagedcheck's terms: a score is a sum of d exact products for each of Q's
three parts, so at most 3 d + 8 roundings of 2^-24 of sum |q_i k_i|, and the parts leave at most 2^-20 of the query's largest
value of every q_i, so 2^-20 max|q| sum |k_i| more. A weight by itself (a mass) has the exponential's 2^-22 and the sum's n 2^-24
beside the score's error.
"""

from __future__ import annotations

import numpy as np

import notcute_flash as nc
from pagedcheck import View, decode_bits, encode, make_table  # noqa: F401

VALUES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6])
LEAST, MOST = {"f16": 104, "bf16": 2}, {"f16": 140, "bf16": 252}


def quantise(x, dtype):
    """Codes [..., d] and scale bytes [..., d / 32] of float64 rows, by the header's words."""
    g = np.asarray(x, dtype=np.float64).reshape(*x.shape[:-1], -1, 32)
    top = np.abs(g).max(-1)
    bad = ~np.isfinite(top)
    top = np.where(bad, 0.0, top)
    k = np.full(top.shape, LEAST[dtype] - 127)
    for e in range(LEAST[dtype] - 127, MOST[dtype] - 127):  # the least k with max <= 7 2^k
        k = np.where(top > 7 * 2.0 ** e, e + 1, k)
    y = np.where(bad[..., None], 0.0, g) / (2.0 ** k)[..., None]
    d = np.abs(np.minimum(np.abs(y), 6.0)[..., None] - VALUES[:8])
    best = d.min(-1, keepdims=True)
    near = d == best
    first, last = near.argmax(-1), 7 - near[..., ::-1].argmax(-1)
    code = np.where((first != last) & (first % 2 == 1), last, first)
    code = np.where(bad[..., None], 0, code | np.where(np.signbit(y), 8, 0))
    return code.astype(np.uint8).reshape(x.shape), np.where(bad, 255, k + 127).astype(np.uint8)


def values(codes, scales):
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return VALUES[codes] * np.repeat(s, 32, axis=-1)


class Pool4:
    """K and V codes and scales of one layout, filled with quantised noise (or, `poison`, groups of NaN)."""

    def __init__(self, rng, pages, heads, ps, d, dtype="f16", layout="hnd", pad=0, poison=False):
        self.pages, self.heads, self.ps, self.d, self.dtype = pages, heads, ps, d, dtype
        row = d + pad
        if layout == "hnd":
            self.strides = (heads * ps * row + pad, ps * row, row)
        elif layout == "nhd":
            self.strides = (ps * heads * row + pad, row, heads * row)
        else:  # K and V of a token next to each other in one allocation
            self.strides = (ps * heads * 2 * row, 2 * row, 2 * heads * row)
        self.gap = row if layout == "inter" else 0
        self.len = (pages - 1) * self.strides[0] + (heads - 1) * self.strides[1] + (ps - 1) * self.strides[2] + d
        n = self.len + self.gap
        self.codes, self.scales = [], []  # one value each
        for _ in range(1 if self.gap else 2):
            if poison:
                c, s = rng.integers(0, 16, n).astype(np.uint8), np.full(n // 32, 255, np.uint8)
            else:
                c, s = quantise(rng.standard_normal((n // 32, 32)), dtype)
                c, s = c.ravel(), s.ravel()
            self.codes.append(c)
            self.scales.append(s)

    def _at(self, page, head, tok):
        page, head, tok = (np.asarray(x, dtype=np.int64) for x in (page, head, tok))
        return page * self.strides[0] + head * self.strides[1] + tok * self.strides[2]

    def get(self, which, page, head, tok):
        """Values in float64."""
        at = self._at(page, head, tok) + which * self.gap
        i = 0 if self.gap else which
        return values(self.codes[i][at[..., None] + np.arange(self.d)], self.scales[i][at[..., None] // 32 + np.arange(self.d // 32)])

    def put(self, which, page, head, tok, codes, scales):
        at = self._at(page, head, tok) + which * self.gap
        i = 0 if self.gap else which
        self.codes[i][at[..., None] + np.arange(self.d)] = codes
        self.scales[i][at[..., None] // 32 + np.arange(self.d // 32)] = scales

    def put_values(self, which, page, head, tok, x):
        self.put(which, page, head, tok, *quantise(x, self.dtype))

    def options(self):
        return dict(head_dim=self.d, page_size=self.ps, num_pages=self.pages, num_kv_heads=self.heads, dtype=self.dtype,
                    page_stride=self.strides[0], head_stride=self.strides[1], token_stride=self.strides[2])

    def upload(self):
        """(K codes, V codes, K scales, V scales): views where K and V are interleaved."""
        codes = [nc.DeviceBuffer.from_array(c[0::2] | (c[1::2] << 4)) for c in self.codes]
        scales = [nc.DeviceBuffer.from_array(s) for s in self.scales]
        if self.gap:
            return codes[0], View(codes[0], self.gap // 2), scales[0], View(scales[0], self.gap // 32)
        return (*codes, *scales)

    def download(self, bufs):
        """(codes, scales) as the pool holds them."""
        out = []
        for i in range(len(self.codes)):
            b = bufs[i].download(np.uint8, self.codes[i].size // 2)
            out.append(np.stack([b & 15, b >> 4], axis=1).ravel())
        return out, [bufs[2 + i].download(np.uint8, self.scales[i].size) for i in range(len(self.scales))]


def rows_of(pool, table, lens, r, which, h):
    """Values of request r's tokens of one head that are in the pool, in float64, and their places."""
    n = min(max(int(lens[r]), 0), table.shape[1] * pool.ps)
    pos = np.arange(n)
    page = table[r, pos // pool.ps].astype(np.int64) if n else np.zeros(0, np.int64)
    here = (page >= 0) & (page < pool.pages)
    x = pool.get(which, page[here], h, (pos % pool.ps)[here])
    return (x if x.dtype == np.float64 else decode_bits(x, pool.dtype)), pos[here]


def ref_attention(q, pool, table, lens, scale, group, four):
    """(o, bound of o, mass added, bound of it) in float64; the masses are [R, tokens of a table row]."""
    R, Hq, d = q.shape
    room = table.shape[1] * pool.ps
    out, bound, mass, mbound = np.zeros((R, Hq, d)), np.zeros((R, Hq, d)), np.zeros((R, room)), np.zeros((R, room))
    qf, scale = decode_bits(q, pool.dtype), float(np.float32(scale))
    for r in range(R):
        for h in range(pool.heads):
            k, pos = rows_of(pool, table, lens, r, 0, h)
            v, _ = rows_of(pool, table, lens, r, 1, h)
            if len(pos) == 0:
                continue
            for i in range(h * group, (h + 1) * group):
                s = scale * (k @ qf[r, i])
                p = np.exp(s - s.max())
                p /= p.sum()
                sums = np.max(np.abs(k) @ np.abs(qf[r, i]))
                ds = abs(scale) * (sums * ((3 * d + 8) if four else (d + 4)) * 2.0 ** -24)
                if four:
                    ds += abs(scale) * 2.0 ** -20 * np.abs(qf[r, i]).max() * np.abs(k).sum(1).max()
                out[r, i] = p @ v
                mag = p @ np.abs(v)
                bound[r, i] = mag * (2 * ds + 2.0 ** -16 + len(pos) * 2.0 ** -24) + np.abs(out[r, i]) * 2.0 ** -23
                mass[r, pos] += p
                mbound[r, pos] += p * (2 * ds + 2.0 ** -22 + (len(pos) + Hq + 2) * 2.0 ** -24)
    return out, bound + 1e-30, mass, mbound + 1e-30


def order_key(x):
    """Masses as Python sorts them: both zeros alike, a NaN above all."""
    return (1, 0.0) if np.isnan(x) else (0, float(x) + 0.0)


def ref_evict(lens, mass, table, free, cursor, ps, room, rules):
    """nc_paged_evict with Python integers: (kept lists by request (None where none is evicted), lens, mass, free, counts)."""
    limit, budget, sinks, recent = rules
    mass, free = mass.copy(), free.copy()
    out, kept, back, dropped, cuts = [], [], [], 0, 0
    for r, n in enumerate(lens.tolist()):
        n = min(max(n, 0), room)
        if n <= limit:
            out.append(n)
            kept.append(None)
            continue
        heavy = sorted(range(sinks, n - recent), key=lambda j: (tuple(-x for x in order_key(mass[r, j])), j))
        keep = list(range(sinks)) + sorted(heavy[:budget - sinks - recent]) + list(range(n - recent, n))
        assert len(keep) == budget
        kept.append(keep)
        mass[r, :n] = np.concatenate([mass[r, keep], np.zeros(n - budget, np.float32)])
        back += table[r, -(-budget // ps):-(-n // ps)].tolist()
        out.append(budget)
        dropped += n - budget
        cuts += 1
    base = int(cursor) - len(back)
    for i, page in enumerate(back):
        if 0 <= base + i < len(free):
            free[base + i] = page
    return kept, np.array(out, np.int32), mass, free, np.array([max(base, 0), cuts, len(back), dropped], np.int32)
