"""Performance cases of a smaller paged cache: fewer bits a value, fewer tokens a request. What a serving program
with long contexts has this library do beside the operators of the 16-bit cache, each operator for itself.

  store   new K and V rows into pages of 4 bits (paged4_append), and back as dense rows (paged4_read), as for a
          prompt that goes on behind a cached one
  decode  attention of one new token per request over pages of 4 bits (paged4_decode)
  mass    attention of one new token per request, and every cached token's share of its weights added up
          (paged_decode_mass over 16 bits, paged4_decode over 4)
  evict   requests that are too long keep their first, their last and their heaviest tokens, moved together in
          their order; the pages that become free go back to the list (paged_evict, paged4_evict)

A case has "op", and of these what its operator needs:
  seqs                   requests
  q_heads, kv_heads, head_dim, dtype ("f16" | "bf16")
  bits                   of the cache: 16 or 4
  page_size, layout      "hnd": a page holds its heads one after the other, "nhd": its tokens
  max_len, lens          cached tokens of the longest request; "even": all the same, "ragged": spread over
                         their logarithm, some requests empty
  rows, pad, source      store: new rows, the share of them that is padding (slot -1), and how K and V
                         stand: "packed", or "fused" (slices of one QKV product's output), or "odd"
                         (rows off 16-byte alignment)
  sigma                  standard deviation of Q (1: ordinary logits, 4: sharp ones)
  limit, budget, sinks, recent   evict: requests longer than limit keep budget tokens, the first `sinks` and the
                         last `recent` always among them
  ties                   evict: masses of few different values
"""

import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
# Scales 2^(byte - 127) that a cache of this type's rows has: the least with values no finer than f16's steps or
# bf16's normal numbers, the largest with values that the type holds.
SCALES = {"f16": (104, 140), "bf16": (2, 252)}
GROUP = 32  # values that share a scale


def _store(name, rows, kv_heads, head_dim, dtype, page_size, layout="hnd", pad=0.0, source="packed"):
    return {"name": name, "op": "store", "rows": rows, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype,
            "page_size": page_size, "layout": layout, "pad": pad, "source": source}


def _decode(name, seqs, q_heads, kv_heads, head_dim, dtype, page_size, max_len, lens, layout="hnd", sigma=1.0, op="decode",
            bits=4):
    return {"name": name, "op": op, "bits": bits, "seqs": seqs, "q_heads": q_heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "dtype": dtype, "page_size": page_size, "max_len": max_len, "lens": lens,
            "layout": layout, "sigma": sigma}


def _evict(name, seqs, kv_heads, head_dim, dtype, page_size, max_len, lens, limit, budget, sinks, recent, layout="hnd",
           ties=False, bits=16):
    return {"name": name, "op": "evict", "bits": bits, "seqs": seqs, "kv_heads": kv_heads, "head_dim": head_dim,
            "dtype": dtype, "page_size": page_size, "max_len": max_len, "lens": lens, "limit": limit, "budget": budget,
            "sinks": sinks, "recent": recent, "layout": layout, "ties": ties}


def listed():
    return [
        # The rows of one decoding step of a small batch.
        _store("store_step", 16, 8, 128, "bf16", 16),
        # Long prompts at once, rows off 16-byte alignment, pages that are no power of two.
        _store("store_prompts_odd", 30000, 8, 64, "f16", 24, pad=0.02, source="odd"),
        # The smallest call: one short request, every head with keys of its own.
        _decode("decode_tiny", 1, 8, 8, 64, "f16", 16, 100, "even"),
        # A batch of chats, four query heads to a key head.
        _decode("decode_chats", 16, 32, 8, 128, "bf16", 16, 1000, "even"),
        # One long document, sharp logits, token-major pages.
        _decode("decode_long", 1, 32, 8, 64, "f16", 64, 120001, "even", layout="nhd", sigma=4.0),
        # A ragged batch of small heads, pages of an odd size.
        _decode("decode_ragged_odd", 33, 16, 4, 32, "f16", 7, 2047, "ragged"),
        # The largest: a full batch of long requests, eight query heads to a key head.
        _decode("decode_large", 96, 64, 8, 128, "bf16", 32, 8192, "even"),
        # A decoding step over a 16-bit cache that keeps count of its tokens' weights.
        _decode("mass_chats", 16, 32, 8, 128, "bf16", 16, 4096, "even", op="mass", bits=16),
        # The same over a ragged batch in 4 bits.
        _decode("mass_ragged", 64, 32, 4, 64, "bf16", 16, 16000, "ragged", op="mass", bits=4),
        # One short chat, cut when it has grown past its limit.
        _evict("evict_one", 1, 8, 64, "f16", 16, 300, "even", 256, 128, 4, 64),
        # A batch of chats, all cut to half of what they may grow to.
        _evict("evict_batch", 16, 8, 128, "bf16", 16, 4097, "even", 4096, 2048, 4, 512),
        # Long documents of different lengths with many equal masses, pages that are no power of two.
        _evict("evict_long_odd", 6, 4, 64, "f16", 24, 60001, "ragged", 9000, 7001, 16, 1001, layout="nhd", ties=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("store", "decode", "decode", "mass", "evict"))
    page_size = rng.choice((16, 16, 16, 32, 64, 128, 1, 7, 24, 100))
    layout = rng.choice(("hnd", "hnd", "nhd"))
    dtype = rng.choice(("f16", "bf16"))
    head_dim, kv_heads = rng.choice((32, 64, 64, 128, 128)), rng.choice((1, 2, 3, 4, 8, 8, 16, 32))
    if op == "store":
        most = 30000 * 8 * 64 // (head_dim * kv_heads)
        case = _store("", _log(rng, 1, min(most, 60000)), kv_heads, head_dim, dtype, page_size, layout,
                      rng.choice((0.0, 0.0, 0.2)), rng.choice(("packed", "fused", "odd")))
    elif op == "evict":
        seqs, max_len = _log(rng, 1, 64), _log(rng, 64, 60000)
        # rows of the cache in all: at most those of the largest listed case
        max_len = max(64, min(max_len, 16 * 4097 * 8 * 128 // (seqs * kv_heads * head_dim)))
        limit = int(max_len * rng.uniform(0.2, 1.0))
        budget = max(1, int(limit * rng.uniform(0.2, 1.0)))
        sinks = min(budget, rng.choice((0, 4, 16)))
        recent = int((budget - sinks) * rng.choice((0.0, 0.25, 0.5, 1.0)))
        case = _evict("", seqs, kv_heads, head_dim, dtype, page_size, max_len, rng.choice(("even", "ragged")), limit,
                      budget, sinks, recent, layout, rng.choice((False, True)), rng.choice((16, 16, 4)))
    else:
        group = rng.choice((1, 1, 2, 4, 5, 8, 16, 20))
        seqs, max_len = _log(rng, 1, 256), _log(rng, 1, 131072)
        # rows of the cache in all: at most a quarter of the largest listed case's, fewer where weights are kept
        most = 96 * 8192 * 8 * 128 // (4 if op == "decode" else 16)
        max_len = max(1, min(max_len, most // (seqs * kv_heads * head_dim), (1 << 29) // (seqs * kv_heads * group)))
        case = _decode("", seqs, kv_heads * group, kv_heads, head_dim, dtype, page_size, max_len,
                       rng.choice(("even", "ragged")), layout, rng.choice((1.0, 1.0, 4.0)), op,
                       4 if op == "decode" else rng.choice((16, 4)))
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

def _lengths(case, tag="len"):
    """Lengths that depend on the case alone (their order goes by the seed). One request has max_len."""
    rng = random.Random("%s %s" % (tag, sorted((k, v) for k, v in case.items() if k != "name")))
    if case["lens"] == "even":
        return [case["max_len"]] * case["seqs"]
    lens = [0 if rng.random() < 0.06 else _log(rng, 1, case["max_len"]) for _ in range(case["seqs"])]
    lens[0] = case["max_len"]
    return lens


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _quantise(x, dtype):
    """Rows [..., d] in 4 bits: bytes of two values (the first one's in the low half), and a scale byte for every
    32: 2^(byte - 127), the least power with no value above 7 times it. Values 0, 0.5, 1, 1.5, 2, 3, 4, 6 and a
    sign, to nearest, halves to the even code. A group that holds a NaN or an infinity has the scale byte 255."""
    g = x.float().unflatten(-1, (-1, GROUP))
    top = g.abs().amax(-1, keepdim=True)
    lo, hi = SCALES[dtype]
    byte = (((top.view(torch.int32) + 0x1FFFFF) >> 23) - 2).clamp(lo, hi)
    good = torch.isfinite(top)
    y = g.abs() * ((254 - byte) << 23).view(torch.float32)
    code = ((y > 0.25).to(torch.uint8) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5.0))
    code = torch.where(good, code + (torch.signbit(g).to(torch.uint8) << 3), 0).to(torch.uint8).flatten(-2)
    byte = torch.where(good, byte, 255).to(torch.uint8).squeeze(-1)
    return code[..., 0::2] | (code[..., 1::2] << 4), byte


def _values(codes, scales):
    """What bytes of two 4-bit values and their scales stand for, in f32."""
    of = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=codes.device)
    of = torch.cat([of, -of])
    of = torch.stack([of.repeat(16), of.repeat_interleave(16)], dim=1)  # by byte: low half, high half
    x = of[codes.int()].flatten(-2).unflatten(-1, (-1, GROUP))
    scale = (scales.int() << 23).view(torch.float32)
    return (x * torch.where(scales == 255, float("nan"), scale)[..., None]).flatten(-2)


def _rows_in_pages(case, pages, x):
    """[pages, kv_heads, page_size, n] as a view of memory of the case's layout."""
    return x if case["layout"] == "hnd" else x.transpose(1, 2).contiguous().transpose(1, 2)


def _cache(case, pages, gen):
    """K and V pages as [pages, kv_heads, page_size, head_dim] views of their layout, filled; in 4 bits bytes and
    scales of them."""
    shape = (pages, case["kv_heads"], case["page_size"], case["head_dim"])
    out = {}
    for n in "kv":
        x = torch.empty(shape, dtype=DTYPES[case["dtype"]], device="cuda").normal_(generator=gen)
        if case.get("bits", 4) == 16:
            out[n] = _rows_in_pages(case, pages, x)
        else:
            per = max(1, (1 << 27) // (x.numel() // pages))  # pages at a time
            parts = [_quantise(x[i:i + per], case["dtype"]) for i in range(0, pages, per)]
            out[n], out[n + "_scales"] = (_rows_in_pages(case, pages, torch.cat(p)) for p in zip(*parts))
    return out


def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _prepare_store(case, seed):
    gen = _generator(seed)
    rows, h, d, ps = case["rows"], case["kv_heads"], case["head_dim"], case["page_size"]
    pages = -(-rows // ps) + 4
    state = _cache(case, pages, gen)
    # requests' rows stand in consecutive places of pages that are anywhere in the pool
    order = torch.randperm(pages, generator=gen, device="cuda")
    at = torch.arange(rows, device="cuda") + ps // 2
    slots = order[at // ps] * ps + at % ps
    padding = torch.rand(rows, generator=gen, device="cuda") < case["pad"]
    padding[0] = False
    state["slots"] = torch.where(padding, -1, slots).to(torch.int32)
    wide = {"packed": h * d, "fused": 6 * h * d, "odd": h * d + 3}[case["source"]]
    n = 1 if case["source"] == "fused" else 2
    x = [torch.empty(rows * wide + 8, dtype=DTYPES[case["dtype"]], device="cuda").normal_(generator=gen) for _ in range(n)]
    if case["source"] == "fused":  # rows of [q (four query heads to each key head), k, v]
        new = [x[0][i * h * d:] for i in (4, 5)]
    else:
        new = [y[1:] if case["source"] == "odd" else y for y in x]
    state["k_rows"], state["v_rows"] = (y.as_strided((rows, h, d), (wide, d, 1)) for y in new)
    state["k_back"], state["v_back"] = (torch.zeros(rows, h, d, dtype=x[0].dtype, device="cuda") for _ in "kv")
    state["pages"] = pages
    return state


def _prepare_pages(case, seed, gen):
    """A batch's cache, table and lengths: pages anywhere in the pool."""
    lens = _lengths(case)
    random.Random(seed).shuffle(lens)
    ps = case["page_size"]
    width = -(-case["max_len"] // ps)
    held = torch.tensor([-(-n // ps) for n in lens], device="cuda")
    pages = int(held.sum()) + 4
    state = _cache(case, pages, gen)
    order = torch.randperm(pages, generator=gen, device="cuda")
    first = torch.cumsum(held, 0) - held
    cols = torch.arange(width, device="cuda")[None, :]
    table = torch.where(cols < held[:, None], order[(first[:, None] + cols).clamp(max=pages - 1)], -1)
    state.update(table=table.to(torch.int32), lens=_int(lens), pages=pages, order=order, held=int(held.sum()))
    return state


def _prepare_decode(case, seed):
    gen = _generator(seed)
    state = _prepare_pages(case, seed, gen)
    q = torch.empty(case["seqs"], case["q_heads"], case["head_dim"], device="cuda").normal_(generator=gen)
    state["q"] = (q * case["sigma"]).to(DTYPES[case["dtype"]])
    state["scale"] = 1.0 / math.sqrt(case["head_dim"])
    state["o"] = torch.zeros(case["seqs"], case["q_heads"], case["head_dim"], device="cuda")
    if case["op"] == "mass":  # what earlier steps have added
        room = state["table"].shape[1] * case["page_size"]
        state["mass"] = torch.empty(case["seqs"], room, device="cuda").normal_(generator=gen).exp_()
    return state


def _prepare_evict(case, seed):
    gen = _generator(seed)
    state = _prepare_pages(case, seed, gen)
    # weights of a softmax added up: a few tokens have most of it
    room = state["table"].shape[1] * case["page_size"]
    mass = torch.empty(case["seqs"], room, device="cuda").normal_(generator=gen).mul_(2.0).exp_()
    state["mass"] = torch.floor(mass * 4) if case["ties"] else mass
    # the list that pages come off: those of the requests were its first ones
    state["free"] = state.pop("order").to(torch.int32)
    state["cursor"], state["counts"] = _int([state["held"]]), _int([0] * 4)
    state["new_lens"] = _int([0] * case["seqs"])
    if case["bits"] == 4:  # the places of the tokens that may be kept, to read them back by
        ps, most = case["page_size"], max(min(x, case["budget"] if x > case["limit"] else x) for x in _lengths(case))
        at = torch.arange(max(most, 1), device="cuda")
        page = state["table"][:, at // ps]
        seen = at < torch.where(state["lens"] > case["limit"], case["budget"], state["lens"])[:, None]
        state["slots"] = torch.where(seen, page * ps + at % ps, -1).to(torch.int32).flatten()
        shape = (state["slots"].numel(), case["kv_heads"], case["head_dim"])
        state["k_back"], state["v_back"] = (torch.zeros(shape, dtype=DTYPES[case["dtype"]], device="cuda") for _ in "kv")
    return state


def _options(nc, case, state):
    """The options of a cache of this case, with the strides of the tensors that the state holds."""
    k, four = state["k"], 1 if case.get("bits", 4) == 16 else 2  # values of an element of k
    more = {"page_stride": four * k.stride(0), "head_stride": four * k.stride(1), "token_stride": four * k.stride(2)}
    if case["op"] == "store":
        more.update(row_stride=state["k_rows"].stride(0))
    return nc.paged_options(num_seqs=case.get("seqs", 1), num_q_heads=case.get("q_heads", case["kv_heads"]),
                            num_kv_heads=case["kv_heads"], head_dim=case["head_dim"], page_size=case["page_size"],
                            num_pages=state["pages"], max_pages=state["table"].shape[1] if "table" in state else 1,
                            dtype=case["dtype"], **more)


def _plan(state):
    """What a program keeps beside its tensors: options, buffer objects and a zeroed workspace."""
    nc, _ = _library()
    case = state["case"]
    opts = state["opts"] = _options(nc, case, state)
    back = state["back_opts"] = nc.PagedOptions.from_buffer_copy(opts)
    back.row_stride = 0  # rows that are read back are packed
    need = 0
    if case["op"] == "decode":
        need = nc.paged4_workspace_bytes(opts)
    elif case["op"] == "mass":
        need = nc.paged_mass_workspace_bytes(opts) if case["bits"] == 16 else nc.paged4_workspace_bytes(opts, mass=True)
    elif case["op"] == "evict":
        need = nc.paged_evict_workspace_bytes(opts)
        state["rules"] = nc.evict_rules(limit=case["limit"], budget=case["budget"], sinks=case["sinks"], recent=case["recent"])
    state["work"] = torch.zeros(max(need, 16), dtype=torch.uint8, device="cuda")
    state["buffers"] = {n: _Buffer(t) for n, t in state.items() if isinstance(t, torch.Tensor)}


def prepare(case, seed):
    state = {"store": _prepare_store, "decode": _prepare_decode, "mass": _prepare_decode,
             "evict": _prepare_evict}[case["op"]](case, seed)
    state["case"] = case
    if own:
        _plan(state)
    return state


# -- one pass -------------------------------------------------------------------------------------

def _read_back(s):
    """K's and V's rows at the slots, as values of the rows' type; zeros where there is no slot."""
    ps, dtype = s["case"]["page_size"], DTYPES[s["case"]["dtype"]]
    at = s["slots"].long().clamp(min=0)
    page, tok = at // ps, at % ps
    seen = (s["slots"] >= 0)[:, None, None]
    k, v = (torch.where(seen, _values(s[n][page, :, tok], s[n + "_scales"][page, :, tok]), 0.0).to(dtype) for n in "kv")
    return [k, v]


def _plain_store(s):
    ps, dtype = s["case"]["page_size"], s["case"]["dtype"]
    # a padding row does once more what the first row does
    at = torch.where(s["slots"] >= 0, s["slots"], s["slots"][0]).long()
    valid = (s["slots"] >= 0)[:, None, None]
    k, v = (_quantise(torch.where(valid, s[n], s[n][:1]), dtype) for n in ("k_rows", "v_rows"))
    s["k"][at // ps, :, at % ps], s["k_scales"][at // ps, :, at % ps] = k
    s["v"][at // ps, :, at % ps], s["v_scales"][at // ps, :, at % ps] = v
    return _read_back(s)


def _gathered(s, n, page, tok):
    """[requests, kv_heads, tokens, head_dim] in f32."""
    x = s[n][page, :, tok].transpose(1, 2)
    return x.float() if s["case"]["bits"] == 16 else _values(x, s[n + "_scales"][page, :, tok].transpose(1, 2))


def _plain_decode(s):
    ps, (seqs, width) = s["case"]["page_size"], s["table"].shape
    d, h = s["case"]["head_dim"], s["case"]["kv_heads"]
    at = torch.arange(width * ps, device="cuda")
    seen = (at[None, :] < s["lens"][:, None])[:, None, :, None]
    page, tok = s["table"].long().clamp(min=0).repeat_interleave(ps, dim=1), (at % ps)[None, :]
    q = s["q"].float().view(seqs, h, -1, d).transpose(2, 3).contiguous()
    scores = torch.matmul(_gathered(s, "k", page, tok), q) * s["scale"]
    scores = torch.where(seen, scores, float("-inf"))
    top = scores.amax(2, keepdim=True)
    p = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
    del scores
    total = p.sum(2)
    v = torch.where(seen, _gathered(s, "v", page, tok), 0.0)
    o = torch.matmul(p.transpose(2, 3).contiguous(), v)
    o = torch.where(total[..., None] > 0, o / total[..., None], 0.0).view(seqs, -1, d)
    if s["case"]["op"] == "decode":
        return o
    s["mass"] += torch.where(seen, p / total[:, :, None, :], 0.0).sum((1, 3))
    return [o, s["mass"]]


def _plain_evict(s):
    c = s["case"]
    ps, (seqs, width), lens = c["page_size"], s["table"].shape, s["lens"].long()
    at = torch.arange(width * ps, device="cuda")[None, :]
    live, cut = at < lens[:, None], (lens > c["limit"])[:, None]
    new = torch.where(lens > c["limit"], c["budget"], lens)
    always = live & ((at < c["sinks"]) | (at >= lens[:, None] - c["recent"]))
    order = torch.sort(torch.where(live & ~always, s["mass"], -1.0), dim=1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(1, order, at.expand(seqs, -1).contiguous())
    keep = live & (always | (rank < c["budget"] - c["sinks"] - c["recent"]) | ~cut)
    to = torch.where(keep, torch.cumsum(keep, 1) - 1, width * ps)
    source = torch.zeros(seqs, width * ps + 1, dtype=torch.long, device="cuda").scatter_(1, to, at.expand(seqs, -1).contiguous())[:, :-1]
    moved = at < new[:, None]
    s["mass"] = torch.where(cut & live, torch.where(moved, s["mass"].gather(1, source), 0.0), s["mass"])
    table = s["table"].long().clamp(min=0)
    # a place that nothing moves to takes its own row; those behind a request's end the row of a page no one has
    spare = s["free"][-1].long()
    from_page, to_page = table.gather(1, source // ps), table.repeat_interleave(ps, dim=1)
    here = torch.where(moved, to_page, spare), torch.where(moved, at % ps, 0)
    there = torch.where(moved, from_page, spare), torch.where(moved, source % ps, 0)
    for n in ("k", "v") if c["bits"] == 16 else ("k", "v", "k_scales", "v_scales"):
        s[n][here[0], :, here[1]] = s[n][there[0], :, there[1]]
    cols = torch.arange(width, device="cuda")[None, :]
    freed = (cols >= ((new + ps - 1) // ps)[:, None]) & (cols < ((lens + ps - 1) // ps)[:, None])
    pages = freed.sum()
    place = s["cursor"].long() - pages + torch.cumsum(freed.flatten(), 0) - 1
    free = torch.cat([s["free"], s["free"][:1]])
    free.scatter_(0, torch.where(freed.flatten(), place, s["free"].numel()), s["table"].flatten())
    s["free"] = free[:-1]
    dropped = torch.where(cut[:, 0], lens - new, 0).sum()
    counts = torch.stack([s["cursor"][0] - pages, cut.sum(), pages, dropped]).to(torch.int32)
    out = [s["mass"], new.to(torch.int32), s["free"], counts]
    return out + ([s["k"], s["v"]] if c["bits"] == 16 else _read_back(s))


def run(state):
    op, bits = state["case"]["op"], state["case"].get("bits", 4)
    if not own:
        return {"store": _plain_store, "decode": _plain_decode, "mass": _plain_decode, "evict": _plain_evict}[op](state)
    nc, module = _library()
    b, opts = state["buffers"], state["opts"]
    if op == "store":
        nc.paged4_append(module, b["k_rows"], b["v_rows"], b["slots"], b["k"], b["v"], b["k_scales"], b["v_scales"], opts)
    elif op == "decode":
        nc.paged4_decode(module, b["q"], b["k"], b["v"], b["k_scales"], b["v_scales"], b["table"], b["lens"], b["o"],
                         b["work"], opts)
        return state["o"]
    elif op == "mass":
        if bits == 16:
            nc.paged_decode_mass(module, b["q"], b["k"], b["v"], b["table"], b["lens"], b["o"], b["mass"], b["work"], opts)
        else:
            nc.paged4_decode(module, b["q"], b["k"], b["v"], b["k_scales"], b["v_scales"], b["table"], b["lens"], b["o"],
                             b["work"], opts, mass=b["mass"])
        return [state["o"], state["mass"]]
    elif bits == 16:
        nc.paged_evict(module, b["table"], b["lens"], b["mass"], b["k"], b["v"], b["free"], b["cursor"], b["new_lens"],
                       b["counts"], b["work"], state["rules"], opts)
    else:
        nc.paged4_evict(module, b["table"], b["lens"], b["mass"], b["k"], b["v"], b["k_scales"], b["v_scales"], b["free"],
                        b["cursor"], b["new_lens"], b["counts"], b["work"], state["rules"], opts)
    out = [state["mass"], state["new_lens"], state["free"], state["counts"]] if op == "evict" else []
    if bits == 16:
        return out + [state["k"], state["v"]]
    nc.paged4_read(module, b["k"], b["v"], b["k_scales"], b["v_scales"], b["slots"], b["k_back"], b["v_back"], state["back_opts"])
    return out + [state["k_back"], state["v_back"]]


def work(case):
    d = case["head_dim"]
    wide, four = case["kv_heads"] * 2 * 2 * d, case["kv_heads"] * 2 * (d // 2 + d // GROUP)  # K and V of a token
    if case["op"] == "store":
        real = case["rows"] * (1 - case["pad"])
        # rows in and their slots, pages written; slots, pages read, rows out
        return {"bytes": real * 2 * (wide + four) + case["rows"] * 8 + (case["rows"] - real) * wide, "flops": 0}
    lens = _lengths(case)
    row = wide if case["bits"] == 16 else four
    if case["op"] == "evict":
        cut = [n for n in lens if n > case["limit"]]
        pages = sum(-(-n // case["page_size"]) for n in cut)
        # masses, the rows that have to move (all but the first ones) read and written; those read back in 4 bits
        bytes_ = sum(cut) * 4 + len(cut) * (case["budget"] - case["sinks"]) * (2 * row + 8) + 4 * pages + 8 * case["seqs"]
        if case["bits"] == 4:
            bytes_ += sum(min(n, case["budget"] if n > case["limit"] else n) for n in lens) * (wide + four + 4)
        return {"bytes": bytes_, "flops": 0}
    entries = sum(-(-n // case["page_size"]) for n in lens)
    qo = case["seqs"] * case["q_heads"] * d * (2 + 4)
    mass = 8 * sum(lens) if case["op"] == "mass" else 0
    return {"bytes": sum(lens) * row + 4 * (entries + case["seqs"]) + qo + mass, "flops": 4 * sum(lens) * case["q_heads"] * d}


# -- the definitions, in 64 bits ------------------------------------------------------------------

def _exact_values(codes, scales):
    """Bytes and scale bytes as float64 values, from the fields of a code: a sign, an exponent and one bit."""
    n = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).double()
    sign, n = torch.where(n >= 8, -1.0, 1.0).double(), n % 8
    e, half = torch.floor(n / 2), n % 2
    x = torch.where(e == 0, half / 2, (1 + half / 2) * torch.pow(2.0, e - 1))
    s = torch.pow(torch.full_like(scales, 2, dtype=torch.float64), scales.double() - 127)
    s = torch.where(scales == 255, float("nan"), s).repeat_interleave(GROUP, dim=-1)
    return sign * x * s


def _exact_store(case, seed):
    s = _prepare_store(case, seed)
    lo, hi = (b - 127 for b in SCALES[case["dtype"]])
    out = []
    for n in ("k_rows", "v_rows"):
        x = s[n].double().reshape(-1, GROUP)
        top = x.abs().amax(1, keepdim=True)
        k = torch.ceil(torch.log2(torch.where(top > 0, top, 2.0 ** lo) / 7)).clamp(lo, hi)
        # log2's last bit: the least k with top <= 7 2^k
        k = torch.where(top <= 7 * torch.pow(2.0, k - 1), k - 1, k)
        k = torch.where(top > 7 * torch.pow(2.0, k), k + 1, k).clamp(lo, hi)
        y = x / torch.pow(2.0, k)
        step = torch.pow(2.0, torch.floor(torch.log2(y.abs().clamp(min=1.0))) - 1)
        y = (torch.round(y / step) * step).clamp(-6.0, 6.0)
        y = torch.where(torch.isfinite(top), y * torch.pow(2.0, k), float("nan")).view(s[n].shape)
        out.append(torch.where((s["slots"] >= 0)[:, None, None], y, 0.0))
    return out


def _exact_rows(case, s, n, pages, i, count):
    """The first `count` rows of head i on these pages."""
    x = s[n][pages, i].flatten(0, 1)[:count]
    return x.double() if case["bits"] == 16 else _exact_values(x, s[n + "_scales"][pages, i].flatten(0, 1)[:count])


def _exact_decode(case, seed):
    s = _prepare_decode(case, seed)
    h, d = case["kv_heads"], case["head_dim"]
    if case["seqs"] * h > 4000:
        return None
    out = torch.zeros(s["o"].shape, dtype=torch.float64, device="cuda")
    mass = s["mass"].double() if "mass" in s else None
    for r, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        pages = s["table"][r, :-(-n // case["page_size"])].long()
        for i in range(h):
            group = slice(i * (case["q_heads"] // h), (i + 1) * (case["q_heads"] // h))
            k, v = (_exact_rows(case, s, x, pages, i, n) for x in "kv")
            p = torch.softmax(torch.matmul(s["q"][r, group].double(), k.t().contiguous()) / math.sqrt(d), dim=1)
            out[r, group] = torch.matmul(p, v)
            if mass is not None:
                mass[r, :n] += p.sum(0)
    return out if mass is None else [out, mass]


def _exact_evict(case, seed):
    s = _prepare_evict(case, seed)
    ps = case["page_size"]
    names = ("k", "v") if case["bits"] == 16 else ("k", "v", "k_scales", "v_scales")
    mass, free, lens = s["mass"].clone(), s["free"].tolist(), s["lens"].tolist()
    table, back, cut, dropped = s["table"].tolist(), [], 0, 0
    for r, n in enumerate(lens):
        if n <= case["limit"]:
            continue
        lo, hi = case["sinks"], n - case["recent"]
        w = mass[r, :n].double().tolist()
        heavy = sorted(range(lo, hi), key=lambda j: (-w[j], j))[:case["budget"] - lo - case["recent"]]
        kept = torch.tensor(list(range(lo)) + sorted(heavy) + list(range(hi, n)), device="cuda")
        pages = s["table"][r].long()
        to = torch.arange(case["budget"], device="cuda")
        for x in names:
            s[x][pages[to // ps], :, to % ps] = s[x][pages[kept // ps], :, kept % ps].clone()
        mass[r, :n] = torch.cat([mass[r, kept], mass.new_zeros(n - case["budget"])])
        back += table[r][-(-case["budget"] // ps):-(-n // ps)]
        lens[r], cut, dropped = case["budget"], cut + 1, dropped + n - case["budget"]
    at = s["held"] - len(back)
    free[at:s["held"]] = back
    out = [mass.double(), _int(lens), _int(free), _int([at, cut, len(back), dropped])]
    if case["bits"] == 16:
        return out + [s["k"].double(), s["v"].double()]
    at = s["slots"].long().clamp(min=0)
    rows = [_exact_values(s[n][at // ps, :, at % ps], s[n + "_scales"][at // ps, :, at % ps]) for n in "kv"]
    return out + [torch.where((s["slots"] >= 0)[:, None, None], x, 0.0) for x in rows]


def exact(case, seed):
    return {"store": _exact_store, "decode": _exact_decode, "mass": _exact_decode, "evict": _exact_evict}[case["op"]](case, seed)
