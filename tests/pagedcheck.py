"""Shared helpers of the paged cache's tests: pools in any layout, references in float64 (and Python
integers), and the error bound of the attention.

Bound of one output element o = sum p_j v_j, p = softmax(s): a score is a sum of d exact products held in
f32 and scaled, so it is off by at most ds = (d + 4) 2^-24 scale sum_i |q_i k_i| (its largest over the
keys); a weight is then off by a factor of 1 + 2 ds, by at most 2^-16 for the exponential, the running
rescales and the split of the weights into two or three 16-bit parts, and n sums in f32 add n 2^-24. All
relative to sum p_j |v_j|, and the final quotient to 2^-23.
"""

from __future__ import annotations

import numpy as np

import notcute_flash as nc

SENTINEL = np.float32(-7777.0)


def decode_bits(bits, dtype):
    if dtype == "bf16":
        return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return bits.view(np.float16).astype(np.float64)


def encode(x, dtype):
    """f32 values to 16-bit patterns, to nearest even."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    if dtype == "bf16":
        u = x.view(np.uint32)
        r = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
        return np.where(np.isnan(x), np.uint16(0x7FC0), r).astype(np.uint16)
    return x.astype(np.float16).view(np.uint16)


class Pool:
    """A K and a V cache of one layout, filled with noise (or NaN where `poison`), with their strides."""

    def __init__(self, rng, pages, heads, ps, d, dtype="f16", layout="hnd", pad=0, poison=False):
        self.pages, self.heads, self.ps, self.d, self.dtype = pages, heads, ps, d, dtype
        row = d + pad
        if layout == "hnd":
            self.strides = (heads * ps * row + pad, ps * row, row)
        elif layout == "nhd":
            self.strides = (ps * heads * row + pad, row, heads * row)
        elif layout == "inter":  # K and V of a token next to each other in one allocation
            self.strides = (ps * heads * 2 * row, 2 * row, 2 * heads * row)
        self.layout = layout
        self.gap = row if layout == "inter" else 0
        self.len = (pages - 1) * self.strides[0] + (heads - 1) * self.strides[1] + (ps - 1) * self.strides[2] + d
        n = self.len + self.gap
        self.bufs = []
        for _ in range(1 if self.gap else 2):
            x = rng.standard_normal(n).astype(np.float32)
            self.bufs.append(encode(np.full(n, np.nan) if poison else x, dtype))

    def index(self, page, head, tok):
        page, head, tok = (np.asarray(x, dtype=np.int64) for x in (page, head, tok))
        at = page * self.strides[0] + head * self.strides[1] + tok * self.strides[2]
        return at[..., None] + np.arange(self.d)

    def get(self, which, page, head, tok):
        buf = self.bufs[0] if self.gap else self.bufs[which]
        return buf[self.index(page, head, tok) + which * self.gap]

    def put(self, which, page, head, tok, bits):
        buf = self.bufs[0] if self.gap else self.bufs[which]
        buf[self.index(page, head, tok) + which * self.gap] = bits

    def options(self):
        return dict(head_dim=self.d, page_size=self.ps, num_pages=self.pages, num_kv_heads=self.heads, dtype=self.dtype,
                    page_stride=self.strides[0], head_stride=self.strides[1], token_stride=self.strides[2])

    def upload(self):
        """(K buffer, V buffer): views of one allocation where K and V are interleaved."""
        dev = [nc.DeviceBuffer.from_array(b) for b in self.bufs]
        if not self.gap:
            return dev[0], dev[1]
        v = View(dev[0], 2 * self.gap)
        return dev[0], v

    def download(self, k, v):
        out = [k.download(np.uint16, self.bufs[0].size)]
        if not self.gap:
            out.append(v.download(np.uint16, self.bufs[1].size))
        return out


class View:
    """The part of a device buffer from an offset on, as a buffer."""

    def __init__(self, base, offset_bytes, nbytes=None):
        self.base = base
        self.ptr = base.ptr + offset_bytes
        self.nbytes = base.nbytes - offset_bytes if nbytes is None else nbytes


def make_table(rng, lens, ps, pages, width, spare=-1):
    """A table of random distinct pages; `spare` where a row's request has none."""
    table = np.full((len(lens), width), spare, dtype=np.int32)
    ids = rng.permutation(pages)
    at = 0
    for r, n in enumerate(lens):
        held = -(-int(max(n, 0)) // ps)
        table[r, :held] = ids[at:at + held]
        at += held
    assert at <= pages
    return table


def ref_decode(q, pool, table, lens, scale, group):
    """(o, bound) in float64: q is [R, Hq, d] bit patterns. Keys on pages outside the pool are absent."""
    R, Hq, d = q.shape
    out, bound = np.zeros((R, Hq, d)), np.zeros((R, Hq, d))
    qf = decode_bits(q, pool.dtype)
    scale = float(np.float32(scale))
    for r in range(R):
        n = min(max(int(lens[r]), 0), table.shape[1] * pool.ps)
        pos = np.arange(n)
        page = table[r, pos // pool.ps].astype(np.int64) if n else np.zeros(0, dtype=np.int64)
        here = (page >= 0) & (page < pool.pages)
        page, tok = page[here], (pos % pool.ps)[here]
        if page.size == 0:
            continue
        for h in range(pool.heads):
            k = decode_bits(pool.get(0, page, h, tok), pool.dtype)
            v = decode_bits(pool.get(1, page, h, tok), pool.dtype)
            for i in range(h * group, (h + 1) * group):
                s = scale * (k @ qf[r, i])
                top = s.max()
                if top == -np.inf:
                    continue
                p = np.exp(s - top)
                p /= p.sum()
                ds = (d + 4) * 2.0 ** -24 * abs(scale) * np.max(np.abs(k) @ np.abs(qf[r, i]))
                out[r, i] = p @ v
                mag = p @ np.abs(v)
                bound[r, i] = mag * (2 * ds + 2.0 ** -16 + page.size * 2.0 ** -24) + np.abs(out[r, i]) * 2.0 ** -23
    return out, bound + 1e-30


def ref_build(cached, new, free, cursor, table, places, ps, num_pages):
    """nc_paged_build with Python integers: (table, lens, offsets, slots, counts)."""
    table = table.copy()
    width = table.shape[1]
    cur = max(int(cursor), 0)
    asked, used, refused, off = cur, 0, 0, 0
    lens, offsets, slots = [], [], np.full(places, -1, dtype=np.int64)
    for r, (c, n) in enumerate(zip(cached.tolist(), new.tolist())):
        c, n = max(c, 0), max(n, 0)
        held, need = -(-c // ps), -(-(c + n) // ps)
        fits = c + n <= width * ps
        take = need - held if fits else 0
        ok = fits and (n == 0 or off + n <= places) and (take == 0 or asked + take <= len(free))
        offsets.append(min(off, places))
        if ok:
            table[r, held:need] = free[asked:asked + take]
            used += take
            for t in range(n):
                page = int(table[r, (c + t) // ps])
                if 0 <= page < num_pages:
                    slots[off + t] = page * ps + (c + t) % ps
        refused += not ok
        lens.append(c + n if ok else c)
        asked += take
        off += n
    offsets.append(min(off, places))
    return (table, np.array(lens, np.int32), np.array(offsets, np.int32), slots.astype(np.int32),
            np.array([cur + used, min(off, places), used, refused], np.int32))
