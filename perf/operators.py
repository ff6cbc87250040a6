"""The operators of a long context served from an 8-bit cache, as a program calls them.

Every case is a dict of plain values. Its "kind" says which operator it takes:

* "rope": rotary positions of the query and key heads of some rows (accel_hip_rope_scaled), in the
  half or the interleaved layout, over part of a head or all of it, with frequencies scaled for a
  long context and positions counted on from a start or given row by row.
* "cache": new keys and values quantised into the 8-bit cache (accel_hip_append_cache_q8: one scale
  for each block of tokens and head, which only grows inside a block) and the touched blocks read
  back (accel_hip_read_cache_q8).
* "read": a range of the 8-bit cache read back alone.
* "attn_q8": causal grouped-query attention over the 8-bit cache (accel_hip_attention_q8), with or
  without a sliding window and its first tokens that stay visible.
* "window": the same with a sliding window over an fp32 cache (accel_hip_attention_window).

`own` is False: the plain form, elementary operations in 32 bits (64 where a quotient is rounded to
a code and for the angles of far positions). `own` is True: the library's calls on the same memory.
"""

import math

import numpy as np
import torch

own = False

THETA = 100000.0
ORIGINAL = 4096  # the context that scaled frequencies were trained at


def listed():
    return [
        # One token's nine query and three key heads: the smallest call, where latency counts.
        {"name": "rope_step_12x64", "kind": "rope", "seq": 1, "heads": 12, "dim": 64, "rotary": 64, "layout": "half",
         "scaling": "none", "position": 2047, "given": False, "extra": 0},
        # A prompt's 32 query and 8 key heads inside the rows of a fused projection, far out, half of each head.
        {"name": "rope_prompt_4096x40x128", "kind": "rope", "seq": 4096, "heads": 40, "dim": 128, "rotary": 64,
         "layout": "interleaved", "scaling": "yarn", "position": 100001, "given": False, "extra": 8},
        # One token into the middle of a block of a small model's cache.
        {"name": "cache_step_3x64", "kind": "cache", "seq": 1, "position": 1037, "kv_heads": 3, "dim": 64, "block": 64},
        # A long prompt into a larger model's cache, from inside a block to inside another.
        {"name": "cache_prompt_4095x8x128", "kind": "cache", "seq": 4095, "position": 100, "kv_heads": 8, "dim": 128,
         "block": 64},
        # A whole context taken back out of the cache, as one does to hand it on.
        {"name": "read_32768x8x128", "kind": "read", "first": 0, "count": 32768, "kv_heads": 8, "dim": 128, "block": 32},
        # A small model's decode step at a full context of 2048.
        {"name": "attn_q8_step_2048", "kind": "attn_q8", "seq": 1, "position": 2047, "heads": 9, "kv_heads": 3,
         "dim": 64, "block": 64, "window": 0, "sinks": 0},
        # A larger model's decode step at the end of a long context.
        {"name": "attn_q8_step_131072", "kind": "attn_q8", "seq": 1, "position": 131071, "heads": 32, "kv_heads": 8,
         "dim": 128, "block": 64, "window": 0, "sinks": 0},
        # Five drafted tokens checked at once, in a window with four tokens that stay visible.
        {"name": "attn_q8_draft_5_window", "kind": "attn_q8", "seq": 5, "position": 20011, "heads": 32, "kv_heads": 8,
         "dim": 128, "block": 16, "window": 8192, "sinks": 4},
        # The next part of a long prompt over what is cached already (the largest product).
        {"name": "attn_q8_prompt_2048", "kind": "attn_q8", "seq": 2048, "position": 4097, "heads": 32, "kv_heads": 8,
         "dim": 128, "block": 64, "window": 0, "sinks": 0},
        # A decode step far out, in a window of 4096.
        {"name": "window_step_4096", "kind": "window", "seq": 1, "position": 30000, "heads": 32, "kv_heads": 8,
         "dim": 128, "window": 4096, "sinks": 4},
        # A prompt of no round length of a small model, from inside a context.
        {"name": "window_prompt_777", "kind": "window", "seq": 777, "position": 5000, "heads": 9, "kv_heads": 3,
         "dim": 64, "window": 512, "sinks": 16},
        # A long prompt of a larger model in a window of 1024.
        {"name": "window_prompt_4096", "kind": "window", "seq": 4096, "position": 0, "heads": 32, "kv_heads": 8,
         "dim": 128, "window": 1024, "sinks": 4},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["rope", "cache", "read", "attn_q8", "attn_q8", "attn_q8", "window", "window"])
    kv = rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([64, 64, 128, 128, 80, 96, 100, 256])
    block = rng.choice([1, 4, 16, 32, 64, 64, 128, 256])
    if kind == "rope":
        heads = kv * rng.choice([2, 3, 4, 5])
        seq = _log_int(rng, 1, max(2, min(8192, 20_000_000 // (heads * dim))))
        return {"kind": kind, "seq": seq, "heads": heads, "dim": dim, "rotary": rng.choice([dim, dim, dim // 2, dim // 4 * 2 - 2]),
                "layout": rng.choice(["half", "interleaved"]),
                "scaling": rng.choice(["none", "linear", "ntk", "yarn", "wavelength"]),
                "position": rng.randrange(0, 1 << rng.randrange(1, 20)), "given": rng.random() < 0.4,
                "extra": rng.choice([0, 0, kv])}
    if kind in ("cache", "read"):
        rows = _log_int(rng, 1, max(2, min(40000, 30_000_000 // (kv * dim))))
        at = rng.randrange(0, 1 << rng.randrange(1, 15))
        if kind == "read":
            return {"kind": kind, "first": at, "count": rows, "kv_heads": kv, "dim": dim, "block": block}
        return {"kind": kind, "seq": min(rows, 8192), "position": at, "kv_heads": kv, "dim": dim, "block": block}
    heads = kv * rng.choice([1, 2, 3, 4, 7])
    seq = 1 if rng.random() < 0.3 else _log_int(rng, 2, 2048)
    windowed = kind == "window" or rng.random() < 0.4
    case = {"kind": kind, "seq": seq, "position": _log_int(rng, 1, max(2, min(131072, 130_000_000 // (kv * dim)))) - 1,
            "heads": heads, "kv_heads": kv, "dim": dim, "block": block,
            "window": _log_int(rng, 1, 8192) if windowed else 0, "sinks": rng.choice([0, 1, 4, 4, 16, 100]) if windowed else 0}
    if kind == "window":
        del case["block"]
    while _pairs(case) * heads * dim > 40e9 or seq * heads * _union(case) > 4e8:
        case["seq"] = seq = max(1, seq // 2)
    return case


# ---- which keys a row sees -----------------------------------------------------------------------

def _rows_seen(case):
    """How many keys each row sees."""
    at = case["position"] + np.arange(case["seq"], dtype=np.int64)
    if not case["window"]:
        return at + 1
    return np.minimum(at + 1, case["window"]) + np.minimum(np.maximum(at + 1 - case["window"], 0), case["sinks"])


def _pairs(case):
    return int(_rows_seen(case).sum())


def _union(case):
    """How many keys some row sees."""
    end = case["position"] + case["seq"]
    low = max(0, case["position"] - case["window"] + 1) if case["window"] else 0
    return end - low + min(low, case["sinks"])


# ---- inputs, made on the GPU from the seed -------------------------------------------------------

def _frequencies(case):
    """Radians per position of each pair, scaled for a context that is 8 times the trained one."""
    r, factor = case["rotary"], 8.0
    i = np.arange(r // 2, dtype=np.float64)
    if case["scaling"] == "ntk" and r > 2:
        return (THETA * factor ** (r / (r - 2))) ** (-2 * i / r)
    f = THETA ** (-2 * i / r)
    if case["scaling"] == "linear":
        return f / factor
    if case["scaling"] == "yarn":
        at = lambda turns: r * math.log(ORIGINAL / (turns * 2 * math.pi)) / (2 * math.log(THETA))  # noqa: E731
        low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), r - 1)
        ramp = np.clip((i - low) / max(high - low, 0.001), 0, 1)
        return f / factor * ramp + f * (1 - ramp)
    if case["scaling"] == "wavelength":
        smooth = np.clip((ORIGINAL * f / (2 * math.pi) - 1) / (4 - 1), 0, 1)
        return f / factor * (1 - smooth) + f * smooth
    return f


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _channels(g, heads, dim):
    """What keys and values look like: some channels are several times larger than others."""
    return torch.exp(0.5 * _normal(g, heads, dim))


def _past(g, rows, heads, dim, block):
    """A filled cache: codes [rows up to a whole block, heads, dim] and scales [blocks, heads]."""
    blocks = -(-rows // block)
    x = (_normal(g, blocks * block, heads, dim) * _channels(g, heads, dim)).view(blocks, block, heads, dim)
    scale = x.abs().amax(dim=(1, 3)) / 127
    codes = torch.round(x / scale[:, None, :, None]).clamp(-127, 127).to(torch.int8)
    return codes.view(blocks * block, heads, dim).contiguous(), scale.contiguous()


def prepare(case, seed):
    kind, g = case["kind"], _generator(seed)
    dim = case["dim"]
    s = {"case": case, "handles": {}}
    if kind == "rope":
        seq, width = case["seq"], (case["heads"] + case["extra"]) * dim
        s["x"] = _normal(g, seq, width)
        s["frequencies"] = torch.from_numpy(_frequencies(case)).cuda()
        s["magnitude"] = 0.1 * math.log(8.0) + 1.0 if case["scaling"] == "yarn" else 1.0
        s["given"] = torch.randint(0, 4096, (seq,), generator=g, device="cuda", dtype=torch.int32) if case["given"] else None
        s["out"] = torch.zeros(seq, width, device="cuda")
        return s
    if kind in ("cache", "read"):
        heads, block = case["kv_heads"], case["block"]
        end = case["position"] + case["seq"] if kind == "cache" else case["first"] + case["count"]
        for name in ("k", "v"):
            s[name + "_codes"], s[name + "_scale"] = _past(g, end, heads, dim, block)
            if kind == "cache":
                s[name] = _normal(g, case["seq"], heads, dim) * _channels(g, heads, dim)
        s["first"] = case["position"] // block * block if kind == "cache" else case["first"]
        s["count"] = end - s["first"]
        for name in ("k", "v"):
            s[name + "_out"] = torch.empty(s["count"], heads, dim, device="cuda")
        return s
    rows, heads = case["position"] + case["seq"], case["kv_heads"]
    s["q"] = 2 * _normal(g, case["seq"], case["heads"], dim)
    s["out"] = torch.empty(case["seq"], case["heads"], dim, device="cuda")
    for name in ("k", "v"):
        if kind == "attn_q8":
            s[name + "_codes"], s[name + "_scale"] = _past(g, rows, heads, dim, case["block"])
        else:
            s[name] = _normal(g, rows, heads, dim) * _channels(g, heads, dim)
    return s


# ---- one pass ------------------------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if kind == "rope":
        return _own_rope(state) if own else _plain_rope(state)
    if kind in ("cache", "read"):
        return _own_cache(state) if own else _plain_cache(state)
    return _own_attention(state) if own else _plain_attention(state)


def _plain_rope(s):
    c = s["case"]
    seq, dim, r = c["seq"], c["dim"], c["rotary"]
    x = s["x"][:, : c["heads"] * dim].reshape(seq, c["heads"], dim)
    at = c["position"] + torch.arange(seq, device="cuda")
    if s["given"] is not None:
        at = c["position"] + s["given"]
    angle = at.double()[:, None] * s["frequencies"][None, :]
    cos, sin = ((f(angle) * s["magnitude"]).float()[:, None, :] for f in (torch.cos, torch.sin))
    if c["layout"] == "half":
        a, b = x[..., : r // 2], x[..., r // 2: r]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).reshape(seq, c["heads"], r)
    return torch.cat([turned, x[..., r:]], dim=-1).reshape(seq, c["heads"] * dim)


def _plain_append(c, x, codes, scale):
    """Rows position .. position + seq of one plane, in place: every touched block's scale is the largest
    magnitude of its new rows over 127, or what it was where rows before them keep more."""
    block, position, seq = c["block"], c["position"], c["seq"]
    b0, b1 = position // block, (position + seq - 1) // block + 1
    kept = position - b0 * block
    rows = torch.zeros((b1 - b0) * block, *x.shape[1:], device="cuda")
    rows[kept:kept + seq] = x
    largest = rows.view(b1 - b0, block, *x.shape[1:]).abs().amax(dim=(1, 3))
    new = largest / torch.full_like(largest, 127)  # a true quotient: a plain number's would be a product
    if kept:
        new[0] = torch.maximum(new[0], scale[b0])
        old = codes[b0 * block:position]
        ratio = scale[b0].double()[None, :, None] / new[0].double()[None, :, None]
        codes[b0 * block:position] = torch.round(old.double() * ratio).nan_to_num(0).to(torch.int8)
    by_row = new.repeat_interleave(block, dim=0)[kept:kept + seq].double()
    codes[position:position + seq] = torch.round(x.double() / by_row[:, :, None]).nan_to_num(0).clamp(-127, 127).to(torch.int8)
    scale[b0:b1] = new


def _plain_cache(s):
    c = s["case"]
    first, end = s["first"], s["first"] + s["count"]
    if c["kind"] == "cache":
        _plain_append(c, s["k"], s["k_codes"], s["k_scale"])
        _plain_append(c, s["v"], s["v_codes"], s["v_scale"])
    at = torch.arange(first, end, device="cuda") // c["block"]
    values = lambda codes, scale: codes[first:end].float() * scale[at][:, :, None]  # noqa: E731
    return {"k": values(s["k_codes"], s["k_scale"]), "v": values(s["v_codes"], s["v_scale"]),
            "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _plain_attention(s):
    c = s["case"]
    seq, heads, kv, dim = c["seq"], c["heads"], c["kv_heads"], c["dim"]
    group, end = heads // kv, c["position"] + seq
    low = max(0, c["position"] - c["window"] + 1) if c["window"] else 0
    keys = torch.cat([torch.arange(min(low, c["sinks"]), device="cuda"), torch.arange(low, end, device="cuda")])
    if c["kind"] == "attn_q8":
        k, v = (s[n + "_codes"][keys].float() * s[n + "_scale"][keys // c["block"]][:, :, None] for n in "kv")
    else:
        k, v = (s[n][keys] for n in "kv")
    q = s["q"].view(seq, kv, group, dim).permute(1, 2, 0, 3).reshape(kv, group * seq, dim)
    scores = torch.matmul(q, k.permute(1, 2, 0).contiguous()) / math.sqrt(dim)
    at = c["position"] + torch.arange(seq, device="cuda")[:, None]
    seen = keys[None, :] <= at
    if c["window"]:
        seen &= (keys[None, :] > at - c["window"]) | (keys[None, :] < c["sinks"])
    scores = scores.view(kv * group, seq, -1).masked_fill_(~seen, -math.inf)
    p = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
    p = (p / p.sum(dim=-1, keepdim=True)).view(kv, group * seq, -1)
    out = torch.matmul(p, v.permute(1, 0, 2).contiguous())
    return out.view(kv, group, seq, dim).permute(2, 0, 1, 3).reshape(seq, heads, dim)


# ---- the library's calls -------------------------------------------------------------------------

def _library():
    from accelep_amd import capi

    return capi, capi.lib()


def _buffer(capi, t):
    return capi.Buffer(t.data_ptr(), t.numel() * t.element_size(), 0) if t is not None else capi.Buffer(None, 0, 0)


def _handle(s, name, make):
    """What a program keeps beside its data: the descriptors of its buffers."""
    if name not in s["handles"]:
        s["handles"][name] = make()
    return s["handles"][name]


def _cache_handle(capi, s):
    c = s["case"]
    return capi.CacheQ8(_buffer(capi, s["k_codes"]), _buffer(capi, s["v_codes"]), _buffer(capi, s["k_scale"]),
                        _buffer(capi, s["v_scale"]), s["k_codes"].shape[0], c["kv_heads"], c["dim"], c["block"])


def _buffers(capi, s, *names):
    return _handle(s, "buffers", lambda: [_buffer(capi, s[n]) for n in names])


def _own_rope(s):
    capi, L = _library()
    c = s["case"]
    x, out, frequencies, given = _buffers(capi, s, "x", "out", "frequencies", "given")
    capi.check(L.accel_hip_rope_scaled(x, out, frequencies, given, c["seq"], c["heads"], c["dim"], s["x"].shape[1],
                                       c["rotary"], capi.ROPE_HALF if c["layout"] == "half" else capi.ROPE_INTERLEAVED,
                                       c["position"], s["magnitude"]))
    return s["out"][:, : c["heads"] * c["dim"]]


def _own_cache(s):
    capi, L = _library()
    c = s["case"]
    cache = _handle(s, "cache", lambda: _cache_handle(capi, s))
    if c["kind"] == "cache":
        k, v, k_out, v_out = _buffers(capi, s, "k", "v", "k_out", "v_out")
        capi.check(L.accel_hip_append_cache_q8(k, v, cache, c["seq"], c["position"], 0))
    else:
        k_out, v_out = _buffers(capi, s, "k_out", "v_out")
    capi.check(L.accel_hip_read_cache_q8(cache, s["first"], s["count"], k_out, v_out))
    return {"k": s["k_out"], "v": s["v_out"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _own_attention(s):
    capi, L = _library()
    c = s["case"]
    if c["kind"] == "attn_q8":
        cache = _handle(s, "cache", lambda: _cache_handle(capi, s))
        q, out = _buffers(capi, s, "q", "out")
        capi.check(L.accel_hip_attention_q8(q, cache, out, c["seq"], c["position"], c["heads"], 0, c["window"],
                                            c["sinks"]))
    else:
        q, k, v, out = _buffers(capi, s, "q", "k", "v", "out")
        capi.check(L.accel_hip_attention_window(q, k, v, out, c["seq"], c["position"], c["heads"], c["kv_heads"],
                                                c["dim"], 0, c["window"], c["sinks"]))
    return s["out"]


# ---- the work of a pass --------------------------------------------------------------------------

def work(case):
    kind, dim = case["kind"], case["dim"]
    if kind == "rope":
        pairs = case["seq"] * case["heads"] * (case["rotary"] // 2)
        return {"bytes": 8 * case["seq"] * case["heads"] * dim + 4 * case["rotary"] + (4 * case["seq"] if case["given"] else 0),
                "flops": 6 * pairs}
    if kind in ("cache", "read"):
        heads, block = case["kv_heads"], case["block"]
        first = case["position"] // block * block if kind == "cache" else case["first"]
        end = case["position"] + case["seq"] if kind == "cache" else case["first"] + case["count"]
        row, scales = heads * dim, 8 * heads * ((end - 1) // block - first // block + 1)
        if kind == "read":  # codes in, values out
            return {"bytes": 2 * row * (end - first) * 5 + scales, "flops": 2 * row * (end - first)}
        # new rows in, their codes and scales out; values of the touched blocks out, older codes of the first in
        new = case["seq"]
        return {"bytes": 2 * row * (5 * new + (end - first - new) + 4 * (end - first)) + 2 * scales,
                "flops": 2 * row * (3 * new + (end - first))}
    rows = case["seq"] * case["heads"] * dim
    keys = _union(case) * case["kv_heads"]
    each = 8 * dim if kind == "window" else 2 * dim + 8 / case["block"]
    return {"bytes": 8 * rows + keys * each, "flops": 4 * _pairs(case) * case["heads"] * dim}


# ---- 64-bit results ------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rope":
        return _exact_rope(case, s)
    if case["kind"] in ("cache", "read"):
        return _exact_cache(case, s)
    return _exact_attention(case, s)


def _exact_rope(c, s):
    """Each pair as a complex number, times e^(i angle)."""
    seq, heads, dim, r = c["seq"], c["heads"], c["dim"], c["rotary"]
    out = s["x"].double()[:, : heads * dim].reshape(seq, heads, dim)
    at = torch.full((seq,), c["position"], device="cuda", dtype=torch.int64)
    at += s["given"].long() if c["given"] else torch.arange(seq, device="cuda")
    turn = torch.polar(torch.full((seq, 1, r // 2), s["magnitude"], device="cuda", dtype=torch.float64),
                       at.double()[:, None, None] * s["frequencies"])
    index = torch.arange(r // 2, device="cuda")
    first, second = (index, index + r // 2) if c["layout"] == "half" else (2 * index, 2 * index + 1)
    z = torch.complex(out[..., first], out[..., second]) * turn
    out[..., first], out[..., second] = z.real, z.imag
    return out.reshape(seq, heads * dim)


def _exact_cache(c, s):
    """Row by row: what a block's scale has to hold, and each value's nearest code."""
    block, got = c["block"], {}
    first, end = s["first"], s["first"] + s["count"]
    for name in ("k", "v"):
        codes, scale = s[name + "_codes"].double(), s[name + "_scale"].double()
        if c["kind"] == "cache":
            at = torch.arange(c["position"], end, device="cuda")
            x, of = s[name].double(), at // block
            need = torch.zeros_like(scale)
            need.index_reduce_(0, of, x.abs().amax(dim=2), "amax", include_self=True)
            need = (need / 127).float().double()  # a scale is held in 32 bits
            here = torch.arange(of[0], of[-1] + 1, device="cuda")
            if c["position"] % block:
                need[of[0]] = torch.maximum(need[of[0]], scale[of[0]])
                codes[first:c["position"]] = torch.round(codes[first:c["position"]] * scale[of[0]][:, None] / need[of[0]][:, None])
            scale[here] = need[here]
            codes[at] = torch.round(x / scale[of][:, :, None])
        rows = torch.arange(first, end, device="cuda")
        got[name], got[name + "_scale"] = codes[rows] * scale[rows // block][:, :, None], scale
    return got


def _exact_attention(c, s):
    seq, heads, kv, dim = c["seq"], c["heads"], c["kv_heads"], c["dim"]
    group, rows = heads // kv, c["position"] + seq
    out = torch.empty(seq, heads, dim, device="cuda", dtype=torch.float64)
    t = torch.arange(rows, device="cuda")
    for h in range(kv):
        if c["kind"] == "attn_q8":
            k, v = (s[n + "_codes"][:rows, h].double() * s[n + "_scale"][:, h].double()[t // c["block"]][:, None] for n in "kv")
        else:
            k, v = (s[n][:rows, h].double() for n in "kv")
        k = k.T.contiguous()
        for s0 in range(0, seq, 512):
            at = c["position"] + torch.arange(s0, min(seq, s0 + 512), device="cuda")[:, None]
            hidden = t[None, :] > at
            if c["window"]:
                hidden |= (at - t[None, :] >= c["window"]) & (t[None, :] >= c["sinks"])
            for q in range(h * group, (h + 1) * group):
                p = (s["q"][s0:s0 + 512, q].double() @ k) / math.sqrt(dim)
                out[s0:s0 + 512, q] = torch.softmax(p.masked_fill(hidden, -math.inf), dim=-1) @ v
    return out
