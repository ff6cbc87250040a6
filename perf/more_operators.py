"""The operators of many requests served together from one cache in pages, as a program calls them.

Every case is a dict of plain values. Its "kind" says which operator it takes:

* "tables": one step's bookkeeping on the GPU (accel_hip_batch_tables): from every request's length and
  new tokens the first row of each request, pages from the free stack for what has no room yet, and each
  new token's position and slot in the cache.
* "append": new keys and values put into their slots (accel_hip_append_paged), in the cache's type.
* "paged": causal grouped-query attention of each request's new tokens over its pages
  (accel_hip_attention_paged): single tokens, chunks of a prompt, both in one call, with or without a window.
* "packed": the same over whole prompts that lie one behind the other, no cache (accel_hip_attention_packed).

`own` is False: the plain form, elementary operations in 32 bits. `own` is True: the library's calls on the
same memory. How long each request is follows from the case alone, what it holds from the seed.
"""

import math

import numpy as np
import torch

own = False

GOLDEN = 0.6180339887498949
TYPES = {"f32": torch.float32, "f16": torch.float16}


def listed():
    return [
        # A decode step of 64 requests: the smallest call, where latency counts.
        {"name": "tables_step_64", "kind": "tables", "requests": 64, "prompts": 0, "chunk_low": 1, "chunk": 1,
         "seen_low": 10, "seen_high": 4000, "page": 16, "pad": 0},
        # A large step: chunks of 40 prompts beside a thousand decoding requests.
        {"name": "tables_mixed_1000", "kind": "tables", "requests": 1000, "prompts": 40, "chunk_low": 100, "chunk": 1500,
         "seen_low": 0, "seen_high": 20000, "page": 64, "pad": 37},
        # One new token of 16 requests of a small model, cache in fp32.
        {"name": "append_step_16x3x64_f32", "kind": "append", "rows": 16, "kv_heads": 3, "dim": 64, "type": "f32",
         "page": 16, "skip": 0, "extra": 9},
        # Chunks of prompts of a larger model, cache in f16; some rows are padding.
        {"name": "append_chunk_8191x8x128_f16", "kind": "append", "rows": 8191, "kv_heads": 8, "dim": 128, "type": "f16",
         "page": 64, "skip": 97, "extra": 0},
        # A small model's decode step with four requests.
        {"name": "paged_step_4_f32", "kind": "paged", "requests": 4, "prompts": 0, "chunk_low": 1, "chunk": 1,
         "seen_low": 100, "seen_high": 2000, "page": 16, "heads": 9, "kv_heads": 3, "dim": 64, "type": "f32",
         "window": 0, "pad": 0},
        # A larger model's decode step, requests of very different lengths.
        {"name": "paged_step_32_f16", "kind": "paged", "requests": 32, "prompts": 0, "chunk_low": 1, "chunk": 1,
         "seen_low": 512, "seen_high": 16384, "page": 64, "heads": 32, "kv_heads": 8, "dim": 128, "type": "f16",
         "window": 0, "pad": 0},
        # Many short requests over an fp32 cache in small pages, the batch padded to a round number of rows.
        {"name": "paged_step_125_f32", "kind": "paged", "requests": 125, "prompts": 0, "chunk_low": 1, "chunk": 1,
         "seen_low": 16, "seen_high": 2048, "page": 16, "heads": 32, "kv_heads": 8, "dim": 128, "type": "f32",
         "window": 0, "pad": 3},
        # Chunks of two long prompts beside 30 decoding requests.
        {"name": "paged_mixed_32_f16", "kind": "paged", "requests": 32, "prompts": 2, "chunk_low": 900, "chunk": 1200,
         "seen_low": 1000, "seen_high": 9000, "page": 64, "heads": 32, "kv_heads": 8, "dim": 128, "type": "f16",
         "window": 0, "pad": 0},
        # Chunks of prompts of a model with a window of 1024, odd lengths, cache in fp32.
        {"name": "paged_chunks_window_f32", "kind": "paged", "requests": 6, "prompts": 6, "chunk_low": 200, "chunk": 500,
         "seen_low": 0, "seen_high": 8000, "page": 32, "heads": 32, "kv_heads": 8, "dim": 128, "type": "f32",
         "window": 1024, "pad": 5},
        # Short prompts of a small model.
        {"name": "packed_24_short", "kind": "packed", "requests": 24, "prompts": 24, "chunk_low": 5, "chunk": 300,
         "heads": 9, "kv_heads": 3, "dim": 64, "window": 0, "fused": True, "pad": 0},
        # A large batch of prompts of a larger model, inside the rows of a fused projection.
        {"name": "packed_7_long", "kind": "packed", "requests": 7, "prompts": 7, "chunk_low": 400, "chunk": 3500,
         "heads": 32, "kv_heads": 8, "dim": 128, "window": 0, "fused": True, "pad": 11},
        # A head for every query, of 80.
        {"name": "packed_3_heads_of_80", "kind": "packed", "requests": 3, "prompts": 3, "chunk_low": 700, "chunk": 2100,
         "heads": 16, "kv_heads": 16, "dim": 80, "window": 0, "fused": False, "pad": 0},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["tables", "append", "paged", "paged", "paged", "paged", "packed", "packed", "packed"])
    page = rng.choice([16, 16, 32, 64, 64, 128, 256])
    kv = rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([64, 64, 128, 128, 128, 80, 96, 100, 256])
    if kind == "append":
        return {"kind": kind, "rows": _log_int(rng, 1, max(2, min(16384, 8_000_000 // (kv * dim)))), "kv_heads": kv,
                "dim": dim, "type": rng.choice(["f32", "f16"]), "page": page, "skip": rng.choice([0, 0, 5, 97]),
                "extra": rng.choice([0, kv, 3 * kv])}
    requests = _log_int(rng, 1, 1000 if kind == "tables" else 128)
    form = rng.choice(["step", "step", "chunks", "mixed"]) if kind != "packed" else "chunks"
    prompts = 0 if form == "step" else requests if form == "chunks" else rng.randrange(1, max(2, requests // 8 + 1))
    chunk = _log_int(rng, 2, 2048) if prompts else 1
    case = {"kind": kind, "requests": requests, "prompts": min(prompts, requests),
            "chunk_low": rng.randrange(1, chunk + 1), "chunk": chunk, "pad": rng.choice([0, 0, 1, 7, 40])}
    if kind != "packed":
        high = _log_int(rng, 1, 32768)
        case.update({"seen_low": rng.randrange(0, high + 1), "seen_high": high, "page": page})
    if kind != "tables":
        case.update({"heads": kv * rng.choice([1, 2, 3, 4, 7]), "kv_heads": kv, "dim": dim,
                     "window": _log_int(rng, 1, 4096) if rng.random() < 0.25 else 0})
        case.update({"type": rng.choice(["f32", "f16", "f16"])} if kind == "paged" else {"fused": rng.random() < 0.5})
    while _too_large(case):
        if case["requests"] > 1:
            case["requests"] = max(1, case["requests"] * 3 // 4)
            case["prompts"] = min(case["prompts"], case["requests"])
        elif case["chunk"] > 2:
            case["chunk"] = case["chunk"] * 3 // 4
            case["chunk_low"] = min(case["chunk_low"], case["chunk"])
        else:
            case["seen_high"] = case["seen_high"] * 3 // 4
            case["seen_low"] = min(case["seen_low"], case["seen_high"])
    return case


def _too_large(case):
    w = work(case)
    if case["kind"] == "tables":
        return _total(case) > 20000
    seen, new = _lengths(case)
    # The plain form's scores, and what one pass of the largest listed case costs.
    return w["flops"] > 1.8e11 or w["bytes"] > 5e8 or case["heads"] * max(n * (s + n) for s, n in zip(seen, new)) > 8e8


# ---- the requests of a case ----------------------------------------------------------------------

def _spread(i, low, high, turn):
    """The i-th of a row of lengths, spread evenly over the logarithm."""
    at = math.modf((i + 1) * GOLDEN + turn)[0]
    return int(round((low + 1) * ((high + 1) / (low + 1)) ** at)) - 1


def _lengths(case):
    """Tokens of each request that are cached already, and its new ones."""
    r = range(case["requests"])
    seen = [_spread(i, case["seen_low"], case["seen_high"], 0.0) if "seen_low" in case else 0 for i in r]
    return seen, [_spread(i, case["chunk_low"], case["chunk"], 0.37) if i < case["prompts"] else 1 for i in r]


def _total(case):
    return sum(_lengths(case)[1])


def _pairs(case):
    """Keys that rows see, over all rows of a head; and keys that some row sees, over all requests."""
    pairs = union = 0
    w = case["window"]
    for s, n in zip(*_lengths(case)):
        at = np.arange(s, s + n, dtype=np.int64) + 1
        pairs += int((np.minimum(at, w) if w else at).sum())
        union += s + n - (max(0, s + 1 - w) if w else 0)
    return pairs, union


# ---- inputs, made on the GPU from the seed -------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _channels(g, heads, dim):
    """What keys and values look like: some channels are several times larger than others."""
    return torch.exp(0.5 * _normal(g, heads, dim))


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pages_of(lengths, page):
    return [-(-n // page) for n in lengths]


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": case, "handles": {}}
    return {"tables": _prepare_tables, "append": _prepare_append, "paged": _prepare_paged,
            "packed": _prepare_packed}[case["kind"]](case, s, g)


def _prepare_tables(case, s, g):
    page = case["page"]
    seen, new = _lengths(case)
    r, rows = len(seen), sum(new) + case["pad"]
    have, need = _pages_of(seen, page), _pages_of([a + b for a, b in zip(seen, new)], page)
    pages, width = sum(need) + 100, max(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)  # which pages who has is chance
    s["table"] = torch.full((r, width), -1, dtype=torch.int32, device="cuda")
    held = torch.arange(width, device="cuda")[None, :] < _ints(have)[:, None]
    s["table"][held] = order[: sum(have)]
    s["stack"] = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
    s["stack"][: pages - sum(have)] = order[sum(have):]
    s["state"] = _ints([pages - sum(have), 0])
    s["counts"], s["lengths"] = _ints(new), _ints(seen)
    s["pages"], s["width"], s["rows"] = pages, width, rows
    for name, n in (("starts", r + 1), ("seen", r), ("slots", rows), ("positions", rows), ("lengths_after", r), ("state_after", 2)):
        s[name] = torch.zeros(n, dtype=torch.int32, device="cuda")
    return s


def _prepare_append(case, s, g):
    rows, page, heads, dim = case["rows"], case["page"], case["kv_heads"], case["dim"]
    pages = -(-2 * rows // page) + 1
    s["pages"] = pages
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:rows].to(torch.int32)
    if case["skip"]:
        slots[case["skip"] - 1:: case["skip"]] = -1
    s["slots"] = slots
    width = (heads + case["extra"]) * dim  # keys, and what else the rows of a projection hold
    scale = torch.cat([_channels(g, heads, dim), torch.ones(case["extra"], dim, device="cuda")]).reshape(width)
    for name in "kv":
        s[name] = _normal(g, rows, width) * scale
        s[name + "_pages"] = torch.zeros(pages, page, heads, dim, dtype=TYPES[case["type"]], device="cuda")
    return s


def _prepare_paged(case, s, g):
    page, heads, kv, dim = case["page"], case["heads"], case["kv_heads"], case["dim"]
    seen, new = _lengths(case)
    rows = sum(new) + case["pad"]
    need = _pages_of([a + b for a, b in zip(seen, new)], page)
    pages, width = sum(need) + 5, max(need) + 2
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    s["table"] = torch.full((len(seen), width), -1, dtype=torch.int32, device="cuda")
    s["table"][torch.arange(width, device="cuda")[None, :] < _ints(need)[:, None]] = order[: sum(need)]
    s["seen"] = _ints(seen)
    s["starts"] = _ints(np.concatenate([[0], np.cumsum(new)]).tolist())
    s["pages"], s["width"], s["rows"] = pages, width, rows
    s["lengths"] = (seen, new)
    s["q"] = 2 * _normal(g, rows, heads, dim)
    s["out"] = torch.zeros(rows, heads, dim, device="cuda")
    for name in "kv":
        c = _channels(g, kv, dim)
        s[name + "_pages"] = torch.empty(pages, page, kv, dim, dtype=TYPES[case["type"]], device="cuda")
        for p in range(0, pages, 4096):
            n = min(4096, pages - p)
            s[name + "_pages"][p:p + n] = _normal(g, n, page, kv, dim) * c
    return s


def _prepare_packed(case, s, g):
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    seen, new = _lengths(case)
    rows = sum(new) + case["pad"]
    s["starts"] = _ints(np.concatenate([[0], np.cumsum(new)]).tolist())
    s["rows"], s["lengths"] = rows, (seen, new)
    q, k, v = 2 * _normal(g, rows, heads, dim), *(_normal(g, rows, kv, dim) * _channels(g, kv, dim) for _ in "kv")
    if case["fused"]:
        whole = torch.cat([q, k, v], dim=1)
        q, k, v = whole[:, :heads], whole[:, heads:heads + kv], whole[:, heads + kv:]
    s["q"], s["k"], s["v"] = q, k, v
    s["out"] = torch.zeros(rows, heads, dim, device="cuda")
    return s


# ---- one pass ------------------------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if kind == "tables":
        return _own_tables(state) if own else _plain_tables(state)
    if kind == "append":
        return _own_append(state) if own else _plain_append(state)
    if kind == "paged":
        return _own_paged(state) if own else _plain_paged(state)
    return _own_packed(state) if own else _plain_packed(state)


def _plain_tables(s):
    page, rows = s["case"]["page"], s["rows"]
    lengths, counts, table = s["lengths"].long(), s["counts"].long(), s["table"]
    have, need = (lengths + page - 1) // page, (lengths + counts + page - 1) // page
    ends, taken = counts.cumsum(0), (need - have).cumsum(0)
    left = s["state"][0].long()
    ok = (taken <= left) | (need == have)
    i = torch.arange(rows, device="cuda")
    of = (i[:, None] >= ends[None, :]).sum(dim=1)  # which request a row is of; past the last one: padding
    padding = of >= len(ends)
    r = of.clamp(max=len(ends) - 1)
    position = torch.where(padding, 0, lengths[r] + i - (ends - counts)[r])
    at = position // page
    fresh = left - 1 - (taken[r] - (need - have)[r] + at - have[r])
    page_id = torch.where(at < have[r], table[r, at].long(), s["stack"][fresh.clamp(0, s["pages"] - 1)].long())
    bad = padding | ~ok[r]
    first = (position % page == 0) & ~padding
    table[r[first], at[first]] = torch.where(ok[r], page_id, -1)[first].to(torch.int32)
    used = torch.where(ok & (need > have), taken, 0).amax()
    return {"starts": torch.cat([torch.zeros_like(ends[:1]), ends]).to(torch.int32), "seen": s["lengths"].clone(),
            "slots": torch.where(bad, -1, page_id * page + position % page).to(torch.int32),
            "positions": position.to(torch.int32), "table": table,
            "lengths_after": torch.where(ok, lengths + counts, lengths).to(torch.int32),
            "state_after": torch.stack([left - used, (~ok).sum()]).to(torch.int32)}


def _plain_append(s):
    c = s["case"]
    n, width = c["rows"], c["kv_heads"] * c["dim"]
    keep = s["slots"] >= 0
    at = s["slots"][keep].long()
    for name in "kv":
        x = s[name][:, :width].reshape(n, c["kv_heads"], c["dim"])
        s[name + "_pages"].view(-1, c["kv_heads"], c["dim"])[at] = x[keep].to(TYPES[c["type"]])
    return {"k": s["k_pages"], "v": s["v_pages"]}


def _plain_attention(c, q, k, v, first, low, out):
    """Rows of one request, the first at position `first`, over its keys from `low` on."""
    n, heads, dim = q.shape
    kv = k.shape[1]
    group = heads // kv
    k = k.permute(1, 2, 0).float().contiguous()
    v = v.permute(1, 0, 2).float().contiguous()
    t = low + torch.arange(k.shape[2], device="cuda")
    for s0 in range(0, n, 1024):
        part = q[s0:s0 + 1024]
        m = part.shape[0]
        x = part.reshape(m, kv, group, dim).permute(1, 2, 0, 3).reshape(kv, group * m, dim)
        scores = torch.matmul(x, k) / math.sqrt(dim)
        if n > 1 or c["window"]:
            at = first + s0 + torch.arange(m, device="cuda")[:, None]
            seen = t[None, :] <= at
            if c["window"]:
                seen &= t[None, :] > at - c["window"]
            scores = scores.view(kv * group, m, -1).masked_fill_(~seen, -math.inf).view(kv, group * m, -1)
        p = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
        p = p / p.sum(dim=-1, keepdim=True)
        out[s0:s0 + m] = torch.matmul(p, v).view(kv, group, m, dim).permute(2, 0, 1, 3).reshape(m, heads, dim)


def _plain_paged(s):
    c = s["case"]
    page, row = c["page"], 0
    k, v = (s[n + "_pages"].view(-1, c["kv_heads"], c["dim"]) for n in "kv")
    for r, (seen, n) in enumerate(zip(*s["lengths"])):
        low = max(0, seen + 1 - c["window"]) if c["window"] else 0
        t = torch.arange(low, seen + n, device="cuda")
        at = s["table"][r, t // page].long() * page + t % page
        _plain_attention(c, s["q"][row:row + n], k[at], v[at], seen, low, s["out"][row:row + n])
        row += n
    return s["out"]


def _plain_packed(s):
    c, row = s["case"], 0
    for n in s["lengths"][1]:
        of = slice(row, row + n)
        _plain_attention(c, s["q"][of], s["k"][of], s["v"][of], 0, 0, s["out"][of])
        row += n
    return s["out"]


# ---- the library's calls -------------------------------------------------------------------------

def _library():
    from accelep_amd import capi

    return capi, capi.lib()


def _buffer(capi, t):
    if t is None:
        return capi.Buffer(None, 0, 0)
    # The bytes from the first value to the last, also of rows that lie apart.
    return capi.Buffer(t.data_ptr(), (1 + sum((n - 1) * d for n, d in zip(t.shape, t.stride()))) * t.element_size(), 0)


def _handle(s, name, make):
    """What a program keeps beside its data: the descriptors of its buffers."""
    if name not in s["handles"]:
        s["handles"][name] = make()
    return s["handles"][name]


def _buffers(capi, s, *names):
    return _handle(s, names, lambda: [_buffer(capi, s[n]) for n in names])


def _batch(capi, s):
    c = s["case"]
    return _handle(s, "batch", lambda: capi.Batch(
        _buffer(capi, s.get("seen")), _buffer(capi, s["starts"]), _buffer(capi, s.get("table")), c["requests"], s["rows"],
        s.get("width", 0), max(_lengths(c)[1])))


def _cache(capi, s):
    c = s["case"]
    return _handle(s, "cache", lambda: capi.CachePaged(
        _buffer(capi, s["k_pages"]), _buffer(capi, s["v_pages"]),
        capi.CACHE_F16 if c["type"] == "f16" else capi.CACHE_F32, s["pages"], c["page"], c["kv_heads"], c["dim"]))


def _own_tables(s):
    capi, L = _library()
    pool = _handle(s, "pool", lambda: capi.PagePool(_buffer(capi, s["stack"]), _buffer(capi, s["state"]), s["pages"],
                                                    s["case"]["page"]))
    counts, lengths, slots, positions, after, state = _buffers(capi, s, "counts", "lengths", "slots", "positions",
                                                               "lengths_after", "state_after")
    capi.check(L.accel_hip_batch_tables(counts, lengths, pool, _batch(capi, s), slots, positions, after, state))
    return {n: s[n] for n in ("starts", "seen", "slots", "positions", "table", "lengths_after", "state_after")}


def _own_append(s):
    capi, L = _library()
    k, v, slots = _buffers(capi, s, "k", "v", "slots")
    capi.check(L.accel_hip_append_paged(k, v, _cache(capi, s), slots, s["case"]["rows"], s["k"].shape[1]))
    return {"k": s["k_pages"], "v": s["v_pages"]}


def _own_paged(s):
    capi, L = _library()
    c = s["case"]
    q, out = _buffers(capi, s, "q", "out")
    capi.check(L.accel_hip_attention_paged(q, _cache(capi, s), _batch(capi, s), out, c["heads"], 0, c["window"]))
    return s["out"]


def _own_packed(s):
    capi, L = _library()
    c = s["case"]
    q, k, v, out = _buffers(capi, s, "q", "k", "v", "out")
    capi.check(L.accel_hip_attention_packed(q, k, v, _batch(capi, s), out, c["heads"], c["kv_heads"], c["dim"],
                                            s["q"].stride(0), s["k"].stride(0), c["window"]))
    return s["out"]


# ---- the work of a pass --------------------------------------------------------------------------

def work(case):
    if case["kind"] == "append":
        values = case["rows"] * case["kv_heads"] * case["dim"]
        return {"bytes": 2 * values * (4 + (2 if case["type"] == "f16" else 4)) + 4 * case["rows"], "flops": 0}
    if case["kind"] == "tables":
        seen, new = _lengths(case)
        r, rows = len(seen), sum(new)
        fresh = sum(_pages_of([a + b for a, b in zip(seen, new)], case["page"])) - sum(_pages_of(seen, case["page"]))
        # counts and lengths in; starts, seen and lengths out; the page each request goes on in; a page's id
        # taken and entered; slots and positions out
        return {"bytes": 4 * (6 * r + 2 * fresh + 2 * (rows + case["pad"])), "flops": 0}
    pairs, union = _pairs(case)
    each = 2 * case["kv_heads"] * case["dim"] * (2 if case.get("type") == "f16" else 4)
    table = 4 * union // case["page"] if "page" in case else 0
    return {"bytes": 8 * _total(case) * case["heads"] * case["dim"] + union * each + table,
            "flops": 4 * pairs * case["heads"] * case["dim"]}


# ---- 64-bit results ------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"tables": _exact_tables, "append": _exact_append, "paged": _exact_attention,
            "packed": _exact_attention}[case["kind"]](case, s)


def _exact_tables(c, s):
    """Token by token, on the host."""
    page, table, stack = c["page"], s["table"].cpu().numpy().copy(), s["stack"].cpu().numpy()
    seen, new = _lengths(c)
    left, refused = int(s["state"][0]), 0
    slots, positions = np.full(s["rows"], -1, np.int32), np.zeros(s["rows"], np.int32)
    starts, after, row = [0], [], 0
    for r, (length, n) in enumerate(zip(seen, new)):
        fresh = -(-(length + n) // page) - -(-length // page)
        room = fresh <= left
        for p in range(length, length + n):
            if p % page == 0:
                table[r, p // page] = stack[left - 1] if room else -1
                left -= 1 if room else 0
            positions[row] = p
            if room:
                slots[row] = table[r, p // page] * page + p % page
            row += 1
        refused += not room
        starts.append(row)
        after.append(length + n if room else length)
    i32 = lambda x: torch.from_numpy(np.asarray(x, np.int32)).cuda()  # noqa: E731
    return {"starts": i32(starts), "seen": i32(seen), "slots": i32(slots), "positions": i32(positions),
            "table": i32(table), "lengths_after": i32(after), "state_after": i32([left, refused])}


def _exact_append(c, s):
    """The nearest value of the cache's type; in 64 bits the caches would be several times larger."""
    out = {}
    for name in "kv":
        pages = s[name + "_pages"].clone().reshape(-1, c["kv_heads"] * c["dim"])
        for i, slot in enumerate(s["slots"].tolist()):
            if slot >= 0:
                pages[slot] = s[name][i, : pages.shape[1]]
        out[name] = pages.reshape(s[name + "_pages"].shape).double()
    return out


def _exact_attention(c, s):
    seen, new = s["lengths"]
    if sum(new) * c["heads"] * max(a + b for a, b in zip(seen, new)) > 4e10:
        return None
    heads, kv, dim = c["heads"], c["kv_heads"], c["dim"]
    group = heads // kv
    out = s["out"].double()
    row = 0
    for r, (length, n) in enumerate(zip(seen, new)):
        for h in range(kv):
            if c["kind"] == "packed":
                k, v = (s[name][row:row + n, h].double() for name in "kv")
            else:
                order = torch.arange(length + n, device="cuda")
                places = s["table"].long()[r][order // c["page"]]
                k, v = (s[name + "_pages"][places, order % c["page"], h].double() for name in "kv")
            order = torch.arange(length + n, device="cuda")[None, :]
            k = k.T.contiguous()
            for s0 in range(0, n, 512):
                m = min(512, n - s0)
                at = length + s0 + torch.arange(m, device="cuda")[:, None]
                hidden = order > at
                if c["window"]:
                    hidden |= at - order >= c["window"]
                x = s["q"][row + s0:row + s0 + m, h * group:(h + 1) * group].double()
                p = torch.matmul(x.permute(1, 0, 2).reshape(group * m, dim), k).view(group, m, -1) / math.sqrt(dim)
                p = torch.softmax(p.masked_fill(hidden, -math.inf), dim=-1).view(group * m, -1)
                out[row + s0:row + s0 + m, h * group:(h + 1) * group] = torch.matmul(p, v).view(group, m, dim).permute(1, 0, 2)
        row += n
    return out
