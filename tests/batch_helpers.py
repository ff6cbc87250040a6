"""Plain forms of what serves a batch of requests from one cache in pages, on the host, and the calls."""

from __future__ import annotations

import ctypes as C

import numpy as np

from accelep_amd import capi
from accelep_amd.capi import Batch, Buffer, CachePaged, PagePool, check, lib
from hip_helpers import dev
from long_context_helpers import NONE, attend

TYPES = {"f32": np.float32, "f16": np.float16}


def ints(values):
    return dev(np.asarray(values, np.int32))


def tables(counts, lengths, table, stack, left, rows, page, pages):
    """One step, token by token: (starts, seen, slots, positions, table, lengths_after, state_after)."""
    table = np.array(table, np.int32)
    slots, positions = np.full(rows, -1, np.int32), np.zeros(rows, np.int32)
    starts, seen, after = [0], [], []
    row = refused = 0
    short = False  # a request got no page: those behind it get none either
    left = min(max(left, 0), pages)
    for r, (count, length) in enumerate(zip(counts, lengths)):
        length = max(int(length), 0)
        n = min(max(int(count), 0), rows - row)
        have, need = -(-length // page), -(-(length + n) // page)
        served = n == 0 or (need <= table.shape[1] and (need == have or (not short and need - have <= left)))
        short = short or (need <= table.shape[1] and not served)
        for p in range(length, length + n):
            if p // page >= have and p % page == 0:
                if served:
                    table[r, p // page] = stack[left - 1]
                    left -= 1
                elif p // page < table.shape[1]:
                    table[r, p // page] = -1
            positions[row] = p
            if served and 0 <= table[r, p // page] < pages:
                slots[row] = table[r, p // page] * page + p % page
            row += 1
        refused += not served
        starts.append(row)
        seen.append(length)
        after.append(length + n if served else length)
    state = [left, refused]
    return {"starts": starts, "seen": seen, "slots": slots, "positions": positions, "table": table,
            "lengths_after": after, "state_after": state}


def released(keep, lengths, table, stack, left, page, pages):
    """(lengths, table, stack, left) after requests are cut to keep[r] tokens."""
    lengths, table, stack = np.array(lengths), np.array(table), np.array(stack)
    for r in range(len(lengths)):
        to, width = max(int(keep[r]), 0), table.shape[1]
        if to >= lengths[r]:
            continue
        for q in range(min(-(-to // page), width), min(-(-int(lengths[r]) // page), width)):
            if 0 <= table[r, q] < pages:
                if left < pages:
                    stack[left] = table[r, q]
                    left += 1
            table[r, q] = -1
        lengths[r] = to
    return lengths, table, stack, left


class Paged:
    """A cache in pages with the requests `seen` + `new` tokens long in it, pages in random order; k and v are the
    tokens' values by request. Everything that no request owns holds `behind`."""

    def __init__(self, rng, seen, new, page, heads, kv_heads, dim, kind, pad=0, extra_pages=3, extra_width=2, behind=np.nan,
                 scale=1.0, longest=None, make=None):
        self.seen, self.new, self.page, self.kind = list(seen), list(new), page, kind
        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        need = [-(-(s + n) // page) for s, n in zip(seen, new)]
        self.pages, self.width, self.rows = sum(need) + extra_pages, max(need, default=0) + extra_width, sum(new) + pad
        order = rng.permutation(self.pages)
        self.table = np.full((len(need), self.width), -1, np.int32)
        self.k, self.v = [], []
        self.planes = {n: np.full((self.pages * page, kv_heads, dim), behind, TYPES[kind]) for n in "kv"}
        used = 0
        for r, pages in enumerate(need):
            self.table[r, :pages] = order[used:used + pages]
            used += pages
            total = self.seen[r] + self.new[r]
            t = np.arange(total)
            at = self.table[r, t // page].astype(np.int64) * page + t % page
            for name, to in (("k", self.k), ("v", self.v)):
                x = (rng.standard_normal((total, kv_heads, dim)) * scale if make is None else make(name, r, total)).astype(TYPES[kind])
                self.planes[name][at] = x
                to.append(x)
        self.starts = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        self.q = (2 * rng.standard_normal((self.rows, heads, dim))).astype(np.float32)
        self.longest = max(new, default=0) if longest is None else longest
        self.upload()

    def upload(self):
        self.d = {"seen": ints(self.seen), "starts": ints(self.starts), "table": ints(self.table),
                  "k": dev(self.planes["k"]), "v": dev(self.planes["v"])}
        self.batch = Batch(self.d["seen"].buffer, self.d["starts"].buffer, self.d["table"].buffer, len(self.seen), self.rows,
                           self.width, self.longest)
        self.cache = CachePaged(self.d["k"].buffer, self.d["v"].buffer, capi.CACHE_F16 if self.kind == "f16" else capi.CACHE_F32,
                                self.pages, self.page, self.kv_heads, self.dim)

    def call(self, window=0, q=None, out=None, row_stride=0):
        qd = dev(self.q) if q is None else q
        out = dev(np.full((self.rows, self.heads, self.dim), 3.0, np.float32)) if out is None else out
        check(lib().accel_hip_attention_paged(qd.buffer, C.byref(self.cache), C.byref(self.batch), out.buffer, self.heads,
                                              row_stride, window))
        return out.numpy()

    def want(self, window=0, rows=None, q=None):
        """(rows, out, bound) of the rows that belong to a request: all, or those of `rows`."""
        q = self.q if q is None else q
        return want_batch(q, self.k, self.v, self.seen, self.starts, window, rows)


def want_batch(q, k, v, seen, starts, window, rows=None):
    at, outs, bounds = [], [], []
    for r in range(len(seen)):
        mine = np.arange(starts[r], starts[r + 1])
        if rows is not None:
            mine = np.intersect1d(mine, rows)
        if len(mine) == 0:
            continue
        out, bound = attend(q[starts[r]:starts[r + 1]], k[r], v[r], seen[r], window, 0, rows=mine - starts[r])
        at.append(mine)
        outs.append(out)
        bounds.append(bound)
    return np.concatenate(at), np.concatenate(outs), np.concatenate(bounds)


def packed_call(q, k, v, starts, heads, kv_heads, dim, rows, window=0, row_stride=0, kv_stride=0, longest=0, requests=None,
                out=None):
    """q, k and v: arrays, or buffers that are there already."""
    held = [x if isinstance(x, Buffer) else dev(np.asarray(x, np.float32)) for x in (q, k, v)]
    qb, kb, vb = (x if isinstance(x, Buffer) else x.buffer for x in held)
    s = ints(starts)
    batch = Batch(NONE, s.buffer, NONE, len(starts) - 1 if requests is None else requests, rows, 0, longest)
    out = dev(np.full((rows, heads, dim), 3.0, np.float32)) if out is None else out
    check(lib().accel_hip_attention_packed(qb, kb, vb, C.byref(batch), out.buffer, heads, kv_heads, dim, row_stride, kv_stride,
                                           window))
    return out.numpy()


def pool_of(stack, left, page):
    held = ints(stack), ints([left, 0])
    return PagePool(held[0].buffer, held[1].buffer, len(stack), page), held
