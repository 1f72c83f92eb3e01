"""Performance cases of the paged key-value cache: what a serving program has this library do in one
decoding step or prompt step, each operator for itself.

  build   block tables, slot map and row offsets from the requests' lengths (paged_build)
  append  the step's new K and V rows into the cache's pages (paged_append)
  decode  attention of one new token per request over its pages (paged_decode)

A case has "op", and of these what its operator needs:
  seqs, width            requests, and the block table's width in pages
  q_heads, kv_heads, head_dim, dtype ("f16" | "bf16")
  page_size, layout      "hnd": a page holds its heads one after the other, "nhd": its tokens
  max_len, lens          cached tokens of the longest request; "even": all the same, "ragged": spread over
                         their logarithm, some requests empty
  new                    new tokens: "one" per request, or up to this many ("ragged", as for prompts)
  rows, pad, source      append: new rows, the share of them that is padding (slot -1), and how K and V
                         stand: "packed", or "fused" (slices of one QKV product's output), or "odd"
                         (rows off 16-byte alignment)
  sigma                  standard deviation of Q (1: ordinary logits, 4: sharp ones)
"""

import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def _build(name, seqs, width, page_size, max_len, new):
    return {"name": name, "op": "build", "seqs": seqs, "width": width, "page_size": page_size, "max_len": max_len,
            "lens": "ragged", "new": new}


def _append(name, rows, kv_heads, head_dim, dtype, page_size, layout="hnd", pad=0.0, source="packed"):
    return {"name": name, "op": "append", "rows": rows, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype,
            "page_size": page_size, "layout": layout, "pad": pad, "source": source}


def _decode(name, seqs, q_heads, kv_heads, head_dim, dtype, page_size, max_len, lens, layout="hnd", sigma=1.0):
    return {"name": name, "op": "decode", "seqs": seqs, "q_heads": q_heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "dtype": dtype, "page_size": page_size, "max_len": max_len, "lens": lens,
            "layout": layout, "sigma": sigma}


def listed():
    return [
        # A decoding step of a small batch: one new token each, now and then a new page.
        _build("build_step", 16, 256, 16, 4000, "one"),
        # A decoding step of a large ragged batch on large pages.
        _build("build_step_many", 1000, 64, 64, 4000, "one"),
        # Prompts admitted together: 256 requests of up to 4096 new tokens.
        _build("build_prompts", 256, 512, 16, 4000, "4096"),
        # The rows of one decoding step of a small batch.
        _append("append_step", 32, 8, 64, "f16", 16),
        # A chunk of prompt rows out of a fused projection's output, bf16, token-major pages.
        _append("append_chunk_fused", 2048, 8, 128, "bf16", 64, layout="nhd", pad=0.1, source="fused"),
        # Long prompts at once, rows off 16-byte alignment, pages that are no power of two.
        _append("append_prompts_odd", 30000, 8, 64, "f16", 24, source="odd"),
        # The smallest call: one short request, every head with keys of its own.
        _decode("decode_tiny", 1, 8, 8, 64, "f16", 16, 100, "even"),
        # A batch of chats, four query heads to a key head.
        _decode("decode_chats", 16, 32, 8, 128, "bf16", 16, 1000, "even"),
        # One long document, sharp logits: the cache's length is the only work there is to split.
        _decode("decode_long", 1, 32, 8, 64, "f16", 64, 120001, "even", layout="nhd", sigma=4.0),
        # A ragged batch with empty places, from one token to thousands.
        _decode("decode_ragged", 64, 32, 4, 64, "bf16", 16, 16000, "ragged"),
        # Small heads with keys of their own, pages of an odd size.
        _decode("decode_heads32_odd", 33, 16, 16, 32, "f16", 7, 2047, "ragged"),
        # The largest: a full batch of long requests, eight query heads to a key head.
        _decode("decode_large", 96, 64, 8, 128, "bf16", 32, 8192, "even"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("build", "append", "decode", "decode", "decode"))
    page_size = rng.choice((16, 16, 16, 32, 64, 128, 1, 7, 24, 100))
    layout = rng.choice(("hnd", "hnd", "nhd"))
    dtype = rng.choice(("f16", "bf16"))
    if op == "build":
        seqs = _log(rng, 1, 2048)
        new = rng.choice(("one", str(_log(rng, 2, 4096))))
        max_len = _log(rng, 1, 4096)
        width = -(-(max_len + 4096) // page_size)
        case = _build("", seqs, min(width, 4096), page_size, max_len, new)
    elif op == "append":
        head_dim, kv_heads = rng.choice((16, 32, 64, 64, 128)), rng.choice((1, 2, 5, 8, 16))
        most = 30000 * 8 * 128 // (head_dim * kv_heads)
        case = _append("", _log(rng, 1, min(most, 60000)), kv_heads, head_dim, dtype, page_size, layout,
                       rng.choice((0.0, 0.0, 0.2)), rng.choice(("packed", "fused", "odd")))
    else:
        head_dim, kv_heads = rng.choice((16, 32, 64, 64, 128, 128)), rng.choice((1, 2, 3, 4, 8, 8, 16, 32))
        group = rng.choice((1, 1, 2, 4, 5, 8, 16, 20))
        seqs, max_len = _log(rng, 1, 256), _log(rng, 1, 131072)
        # rows of the cache in all: at most a quarter of the largest listed case's
        max_len = max(1, min(max_len, 96 * 8192 * 8 * 128 // 4 // (seqs * kv_heads * head_dim)))
        case = _decode("", seqs, kv_heads * group, kv_heads, head_dim, dtype, page_size, max_len,
                       rng.choice(("even", "ragged")), layout, rng.choice((1.0, 1.0, 4.0)))
    del case["name"]
    return case


# -- the library's side ---------------------------------------------------------------------------

_session = None


def _library():
    """The binding and the process's module, made once as a program does at start-up."""
    global _session
    if _session is None:
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "not-cute-zig_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import notcute_flash as nc

        torch.cuda.init()
        nc.init()
        _session = (nc, nc.Module.load_embedded())
    return _session


class _Buffer:
    """A torch tensor as the buffer object the launches take (device address and size)."""

    def __init__(self, tensor):
        self.ptr = tensor.data_ptr()
        self.nbytes = tensor.untyped_storage().nbytes() - tensor.storage_offset() * tensor.element_size()


# -- inputs ---------------------------------------------------------------------------------------

def _lengths(case, tag, most, kind):
    """Lengths that depend on the case alone (their order goes by the seed). One request has `most`."""
    rng = random.Random("%s %s" % (tag, sorted((k, v) for k, v in case.items() if k != "name")))
    if kind == "even":
        return [most] * case["seqs"]
    lens = [0 if rng.random() < 0.06 else _log(rng, 1, most) for _ in range(case["seqs"])]
    lens[0] = most
    return lens


def _build_lengths(case):
    cap = case["width"] * case["page_size"]
    cached = [min(x, cap - 1) for x in _lengths(case, "cached", case["max_len"], case["lens"])]
    if case["new"] == "one":
        new = [1] * case["seqs"]
    else:
        new = _lengths(case, "new", int(case["new"]), "ragged")
    return cached, [min(n, cap - c) for c, n in zip(cached, new)]


def _rows_of(case):
    """Places of the slot map: the new rows, padded to a multiple of 64 as a captured step has them."""
    return -(-sum(_build_lengths(case)[1]) // 64) * 64


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _prepare_build(case, seed):
    rng = random.Random(seed)
    ps, width = case["page_size"], case["width"]
    pairs = list(zip(*_build_lengths(case)))
    rng.shuffle(pairs)
    held = [-(-c // ps) for c, _ in pairs]
    need = sum(-(-(c + n) // ps) for c, n in pairs)
    pages = need + 8
    ids = list(range(pages))
    rng.shuffle(ids)
    table = torch.full((case["seqs"], width), -1, dtype=torch.int32)
    at = 0
    for r, h in enumerate(held):
        table[r, :h] = torch.tensor(ids[at:at + h], dtype=torch.int32)
        at += h
    state = {"cached": _int([c for c, _ in pairs]), "new": _int([n for _, n in pairs]), "free": _int(ids[at:]),
             "cursor": _int([0]), "table": table.cuda(), "pages": pages,
             "lens": _int([0] * case["seqs"]), "offsets": _int([0] * (case["seqs"] + 1)),
             "slots": _int([0] * _rows_of(case)), "counts": _int([0] * 8)}
    return state


def _cache(case, pages, gen):
    """K and V pages as [pages, kv_heads, page_size, head_dim] views of their layout, filled."""
    h, ps, d = case["kv_heads"], case["page_size"], case["head_dim"]
    out = []
    for _ in range(2):
        shape = (pages, h, ps, d) if case["layout"] == "hnd" else (pages, ps, h, d)
        x = torch.empty(shape, dtype=DTYPES[case["dtype"]], device="cuda").normal_(generator=gen)
        out.append(x if case["layout"] == "hnd" else x.transpose(1, 2))
    return out


def _prepare_append(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rows, h, d, ps = case["rows"], case["kv_heads"], case["head_dim"], case["page_size"]
    pages = -(-rows // ps) + 4
    k, v = _cache(case, pages, gen)
    # requests' rows stand in consecutive places of pages that are anywhere in the pool
    order = torch.randperm(pages, generator=gen, device="cuda")
    at = torch.arange(rows, device="cuda") + ps // 2
    slots = order[at // ps] * ps + at % ps
    padding = torch.rand(rows, generator=gen, device="cuda") < case["pad"]
    padding[0] = False
    slots = torch.where(padding, -1, slots).to(torch.int32)
    wide = {"packed": h * d, "fused": 6 * h * d, "odd": h * d + 3}[case["source"]]
    n = 1 if case["source"] == "fused" else 2
    x = [torch.empty(rows * wide + 8, dtype=k.dtype, device="cuda").normal_(generator=gen) for _ in range(n)]
    if case["source"] == "fused":  # rows of [q (four query heads to each key head), k, v]
        new = [x[0][i * h * d:] for i in (4, 5)]
    else:
        new = [y[1:] if case["source"] == "odd" else y for y in x]
    new = [y.as_strided((rows, h, d), (wide, d, 1)) for y in new]
    return {"k_rows": new[0], "v_rows": new[1], "slots": slots, "k": k, "v": v, "pages": pages}


def _prepare_decode(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    lens = _lengths(case, "len", case["max_len"], case["lens"])
    random.Random(seed).shuffle(lens)
    ps = case["page_size"]
    width = -(-case["max_len"] // ps)
    held = torch.tensor([-(-n // ps) for n in lens], device="cuda")
    pages = int(held.sum()) + 4
    k, v = _cache(case, pages, gen)
    order = torch.randperm(pages, generator=gen, device="cuda")
    first = torch.cumsum(held, 0) - held
    cols = torch.arange(width, device="cuda")[None, :]
    table = torch.where(cols < held[:, None], order[(first[:, None] + cols).clamp(max=pages - 1)], -1)
    q = torch.empty(case["seqs"], case["q_heads"], case["head_dim"], device="cuda").normal_(generator=gen)
    q = (q * case["sigma"]).to(DTYPES[case["dtype"]])
    return {"q": q, "k": k, "v": v, "table": table.to(torch.int32), "lens": _int(lens), "pages": pages,
            "scale": 1.0 / math.sqrt(case["head_dim"]),
            "o": torch.zeros(case["seqs"], case["q_heads"], case["head_dim"], device="cuda")}


def _options(nc, case, state):
    """The options of a cache of this case, with the strides of the tensors that the state holds."""
    more = {}
    if case["op"] != "build":
        k = state["k"]
        more = {"page_stride": k.stride(0), "head_stride": k.stride(1), "token_stride": k.stride(2)}
    if case["op"] == "append":
        more.update(row_stride=state["k_rows"].stride(0))
    return nc.paged_options(num_seqs=case.get("seqs", 1), num_q_heads=case.get("q_heads", case.get("kv_heads", 1)),
                            num_kv_heads=case.get("kv_heads", 1), head_dim=case.get("head_dim", 64),
                            page_size=case["page_size"], num_pages=state["pages"],
                            max_pages=state["table"].shape[1] if "table" in state else 1,
                            dtype=case.get("dtype", "f16"), **more)


def prepare(case, seed):
    state = {"build": _prepare_build, "append": _prepare_append, "decode": _prepare_decode}[case["op"]](case, seed)
    state["case"] = case
    if own:
        nc, _ = _library()
        state["opts"] = _options(nc, case, state)
        state["buffers"] = {n: _Buffer(t) for n, t in state.items() if isinstance(t, torch.Tensor)}
        if case["op"] == "decode":
            state["work"] = torch.zeros(nc.paged_workspace_bytes(state["opts"]), dtype=torch.uint8, device="cuda")
            state["buffers"]["work"] = _Buffer(state["work"])
    return state


# -- one pass -------------------------------------------------------------------------------------

def _plain_build(s):
    ps, (seqs, width), places = s["case"]["page_size"], s["table"].shape, s["slots"].shape[0]
    cached, new = s["cached"].long(), s["new"].long()
    held, need = (cached + ps - 1) // ps, (cached + new + ps - 1) // ps
    take = torch.where(need <= width, need - held, 0)
    first = s["cursor"].long() + torch.cumsum(take, 0) - take
    ends = torch.cumsum(new, 0)
    fits = (need <= width) & ((take == 0) | (first + take <= s["free"].shape[0])) & ((new == 0) | (ends <= places))
    cols = torch.arange(width, device=held.device)[None, :]
    mine = fits[:, None] & (cols >= held[:, None]) & (cols < need[:, None])
    from_list = (first[:, None] + cols - held[:, None]).clamp(0, s["free"].shape[0] - 1)
    s["table"] = torch.where(mine, s["free"][from_list], s["table"])
    at = torch.arange(places, device=held.device)
    r = torch.searchsorted(ends, at, right=True).clamp(max=seqs - 1)
    pos = cached[r] + at - (ends - new)[r]
    page = s["table"][r, (pos // ps).clamp(0, width - 1)].long()
    slots = torch.where((at < ends[-1]) & fits[r], page * ps + pos % ps, -1)
    lens = torch.where(fits, cached + new, cached)
    taken = torch.where(fits, take, 0).sum()
    counts = torch.stack([s["cursor"][0] + taken, ends[-1].clamp(max=places), taken, (~fits).sum()])
    offsets = torch.cat([torch.zeros_like(ends[:1]), ends]).clamp(max=places)
    return [s["table"]] + [x.to(torch.int32) for x in (lens, offsets, slots, counts)]


def _plain_append(s):
    ps = s["case"]["page_size"]
    valid = (s["slots"] >= 0)[:, None, None]  # a padding row does once more what the first row does
    slots = torch.where(s["slots"] >= 0, s["slots"], s["slots"][0]).long()
    for rows, cache in ((s["k_rows"], s["k"]), (s["v_rows"], s["v"])):
        cache[slots // ps, :, slots % ps] = torch.where(valid, rows, rows[:1])
    return [s["k"], s["v"]]


def _plain_decode(s):
    ps, (seqs, width) = s["case"]["page_size"], s["table"].shape
    d, h = s["case"]["head_dim"], s["case"]["kv_heads"]
    at = torch.arange(width * ps, device="cuda")
    seen = (at[None, :] < s["lens"][:, None])[:, None, :, None]
    page = s["table"].long().clamp(min=0).repeat_interleave(ps, dim=1)
    k = s["k"][page, :, (at % ps)[None, :]].transpose(1, 2).float()
    q = s["q"].float().view(seqs, h, -1, d).transpose(2, 3).contiguous()
    scores = torch.matmul(k, q) * s["scale"]
    del k
    scores = torch.where(seen, scores, float("-inf"))
    top = scores.amax(2, keepdim=True)
    p = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(2)
    v = s["v"][page, :, (at % ps)[None, :]].transpose(1, 2).float()
    v = torch.where(seen, v, 0.0)
    o = torch.matmul(p.transpose(2, 3).contiguous(), v)
    return torch.where(total[..., None] > 0, o / total[..., None], 0.0).view(seqs, -1, d)


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"build": _plain_build, "append": _plain_append, "decode": _plain_decode}[op](state)
    nc, module = _library()
    b, opts = state["buffers"], state["opts"]
    if op == "build":
        nc.paged_build(module, b["cached"], b["new"], b["free"], b["cursor"], b["table"], b["lens"], b["offsets"],
                       b["slots"], b["counts"], opts)
        return [state["table"], state["lens"], state["offsets"], state["slots"], state["counts"][:4]]
    if op == "append":
        nc.paged_append(module, b["k_rows"], b["v_rows"], b["slots"], b["k"], b["v"], opts)
        return [state["k"], state["v"]]
    nc.paged_decode(module, b["q"], b["k"], b["v"], b["table"], b["lens"], b["o"], b["work"], opts)
    return state["o"]


def work(case):
    if case["op"] == "build":
        cached, new = _build_lengths(case)
        ps = case["page_size"]
        taken = sum(-(-(c + n) // ps) - -(-c // ps) for c, n in zip(cached, new))
        # lengths and offsets, a held page's entry per request, the pages taken (list and table), the slots
        return {"bytes": 4 * (4 * case["seqs"] + case["seqs"] + 2 * taken + _rows_of(case)), "flops": 0}
    row = case["kv_heads"] * case["head_dim"] * 2 * 2
    if case["op"] == "append":
        return {"bytes": case["rows"] * (2 * row * (1 - case["pad"]) + 4), "flops": 0}
    lens = _lengths(case, "len", case["max_len"], case["lens"])
    entries = sum(-(-n // case["page_size"]) for n in lens)
    qo = case["seqs"] * case["q_heads"] * case["head_dim"] * (2 + 4)
    return {"bytes": sum(lens) * row + 4 * (entries + case["seqs"]) + qo,
            "flops": 4 * sum(lens) * case["q_heads"] * case["head_dim"]}


# -- the definitions, in 64 bits ------------------------------------------------------------------

def _exact_build(case, seed):
    s = _prepare_build(case, seed)
    ps, (seqs, width), places = case["page_size"], s["table"].shape, s["slots"].shape[0]
    cached, new, free = (s[n].tolist() for n in ("cached", "new", "free"))
    table = [row for row in s["table"].tolist()]
    lens, offsets, slots, used, asked, refused = [], [0], [-1] * places, 0, 0, 0
    for r in range(seqs):
        held, need = -(-cached[r] // ps), -(-(cached[r] + new[r]) // ps)
        take = need - held if need <= width else 0
        fits = need <= width and (not take or asked + take <= len(free)) and (
            not new[r] or offsets[-1] + new[r] <= places)
        if fits:
            table[r][held:need] = free[asked:asked + take]
            used += take
            for t in range(new[r]):
                pos = cached[r] + t
                slots[offsets[-1] + t] = table[r][pos // ps] * ps + pos % ps
        asked += take
        refused += not fits
        lens.append(cached[r] + (new[r] if fits else 0))
        offsets.append(min(offsets[-1] + new[r], places))
    return [_int(x) for x in (table, lens, offsets, slots, [used, offsets[-1], used, refused])]


def _exact_append(case, seed):
    s = _prepare_append(case, seed)
    out = []
    for rows, cache in ((s["k_rows"], s["k"]), (s["v_rows"], s["v"])):
        flat = cache.double().transpose(1, 2).flatten(0, 1)  # [slot, head, dim]
        flat[s["slots"][s["slots"] >= 0].long()] = rows[s["slots"] >= 0].double()
        out.append(flat.view(cache.shape[0], cache.shape[2], cache.shape[1], cache.shape[3]).transpose(1, 2))
    return out


def _exact_decode(case, seed):
    s = _prepare_decode(case, seed)
    h, d = case["kv_heads"], case["head_dim"]
    out = torch.zeros(s["o"].shape, dtype=torch.float64, device="cuda")
    for r, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        pages = s["table"][r, :-(-n // case["page_size"])].long()
        for i in range(h):
            group = slice(i * (case["q_heads"] // h), (i + 1) * (case["q_heads"] // h))
            k, v = (s[x][pages, i].reshape(-1, d)[:n].double() for x in "kv")
            scores = torch.matmul(s["q"][r, group].double(), k.t().contiguous()) / math.sqrt(d)
            out[r, group] = torch.matmul(torch.softmax(scores, dim=1), v)
    return out


def exact(case, seed):
    return {"build": _exact_build, "append": _exact_append, "decode": _exact_decode}[case["op"]](case, seed)
