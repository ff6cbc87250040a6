"""What the calls over a batch of requests refuse, and with which status: decided on the host from the arguments
alone, so these tests need no GPU (the pointers are never read)."""

from __future__ import annotations

import ctypes as C

import pytest

from accelep_amd.capi import CACHE_F16, CACHE_F32, Batch, CachePaged, PagePool, lib
from test_long_context_refusals import INVALID, NONE, OVERFLOW, buf, refused

GIB = 1 << 30
REQUESTS, ROWS, WIDTH, PAGES, PAGE, KV, DIM, HEADS = 5, 40, 7, 30, 16, 2, 64, 4

# Where each buffer of a call that works lies, GiB, and its bytes.
PLACES = {"counts": (1, 4 * REQUESTS), "lengths": (2, 4 * REQUESTS), "stack": (3, 4 * PAGES), "state": (4, 8),
          "seen": (5, 4 * REQUESTS), "starts": (6, 4 * (REQUESTS + 1)), "table": (7, 4 * REQUESTS * WIDTH),
          "slots": (8, 4 * ROWS), "positions": (9, 4 * ROWS), "lengths_after": (10, 4 * REQUESTS), "state_after": (11, 8),
          "keep": (12, 4 * REQUESTS), "k_pages": (13, 4 * PAGES * PAGE * KV * DIM), "v_pages": (14, 4 * PAGES * PAGE * KV * DIM),
          "k": (15, 4 * ROWS * KV * DIM), "v": (16, 4 * ROWS * KV * DIM), "q": (17, 4 * ROWS * HEADS * DIM),
          "out": (18, 4 * ROWS * HEADS * DIM)}


class Call:
    """The arguments of every call, any of them changed. A sized buffer is exactly as large as it has to be."""

    def __init__(self, **change):
        self.b = {n: change.pop(n) if n in change else buf(size, at * GIB) for n, (at, size) in PLACES.items()}
        self.x = dict(requests=REQUESTS, rows=ROWS, width=WIDTH, longest=0, pages=PAGES, page=PAGE, kv_heads=KV, dim=DIM,
                      type=CACHE_F32, heads=HEADS, row_stride=0, kv_stride=0, window=0)
        self.x.update(change)
        x, b = self.x, self.b
        self.batch = Batch(b["seen"], b["starts"], b["table"], x["requests"], x["rows"], x["width"], x["longest"])
        self.pool = PagePool(b["stack"], b["state"], x["pages"], x["page"])
        self.cache = CachePaged(b["k_pages"], b["v_pages"], x["type"], x["pages"], x["page"], x["kv_heads"], x["dim"])

    def tables(self):
        b = self.b
        return lib().accel_hip_batch_tables(b["counts"], b["lengths"], C.byref(self.pool), C.byref(self.batch), b["slots"],
                                            b["positions"], b["lengths_after"], b["state_after"])

    def release(self):
        return lib().accel_hip_release_pages(self.b["keep"], self.b["lengths"], C.byref(self.pool), C.byref(self.batch))

    def append(self):
        b, x = self.b, self.x
        return lib().accel_hip_append_paged(b["k"], b["v"], C.byref(self.cache), b["slots"], x["rows"], x["row_stride"])

    def paged(self):
        b, x = self.b, self.x
        return lib().accel_hip_attention_paged(b["q"], C.byref(self.cache), C.byref(self.batch), b["out"], x["heads"],
                                               x["row_stride"], x["window"])

    def packed(self):
        b, x = self.b, self.x
        return lib().accel_hip_attention_packed(b["q"], b["k"], b["v"], C.byref(self.batch), b["out"], x["heads"],
                                                x["kv_heads"], x["dim"], x["row_stride"], x["kv_stride"], x["window"])


BUFFERS = {"tables": ("counts lengths stack state", "seen starts table slots positions lengths_after state_after"),
           "release": ("keep", "lengths table stack state"), "append": ("k v slots", "k_pages v_pages"),
           "paged": ("q k_pages v_pages starts seen table", "out"), "packed": ("q k v starts", "out")}
CALLS = sorted(BUFFERS)
EACH = [(c, n) for c in CALLS for n in " ".join(BUFFERS[c]).split()]


@pytest.mark.parametrize("call,name", EACH)
def test_a_buffer_that_is_missing_too_small_or_not_aligned(call, name):
    at, size = PLACES[name]
    refused(getattr(Call(**{name: NONE}), call)(), "out of range")
    refused(getattr(Call(**{name: buf(size - 1, at * GIB)}), call)(), "out of range")
    refused(getattr(Call(**{name: buf(size, at * GIB + 2)}), call)(),
            "not aligned" if name in ("q", "k", "v", "out", "k_pages", "v_pages") else "out of range")


@pytest.mark.parametrize("call,output,other", [
    (c, o, n) for c in CALLS for o in BUFFERS[c][1].split() for n in " ".join(BUFFERS[c]).split()
    if n != o and {o, n} not in ({"lengths", "lengths_after"}, {"state", "state_after"})])
def test_an_output_over_what_the_call_reads_or_writes(call, output, other):
    at, size = PLACES[other]
    own = PLACES[output][1]
    for begin in (at * GIB, at * GIB + size - 4, at * GIB + 4 - own):
        refused(getattr(Call(**{output: buf(own, begin)}), call)(), "overlap")


def test_lengths_and_state_may_be_themselves_but_not_beside_themselves():
    for name in ("lengths", "state"):
        at, size = PLACES[name]
        for shift in (4, -4):
            refused(Call(**{name + "_after": buf(size, at * GIB + shift)}).tables(), "overlap")


@pytest.mark.parametrize("change,calls,text", [
    (dict(requests=-1), "tables release paged packed", "out of range"), (dict(rows=-1), "tables release paged packed", "out of range"),
    (dict(rows=-1), "append", "negative"), (dict(longest=-1), "tables paged packed", "out of range"),
    (dict(width=-1), "tables release paged", "out of range"), (dict(rows=2 ** 31), "tables append paged packed", "too large"),
    (dict(requests=2 ** 31 - 257), "tables release paged packed", "too large"),
    (dict(width=2 ** 27), "tables release paged", "too wide"), (dict(width=2 ** 62), "tables release paged", "too wide"),
    (dict(page=8), "tables release append paged", "power of two"), (dict(page=0), "tables release append paged", "power of two"),
    (dict(page=48), "tables release append paged", "power of two"), (dict(page=512), "tables release append paged", "power of two"),
    (dict(page=-16), "tables release append paged", "power of two"), (dict(pages=-1), "tables release append paged", "out of range"),
    (dict(pages=0), "append paged", "out of range"), (dict(pages=2 ** 27), "tables release", "out of range"),
    (dict(pages=2 ** 27), "append paged", "too large"), (dict(type=2), "append paged", "type"), (dict(type=-1), "append paged", "type"),
    (dict(kv_heads=0), "append paged packed", "out of range"), (dict(kv_heads=-2), "append paged packed", "out of range"),
    (dict(dim=0), "append paged packed", "out of range" ), (dict(dim=257), "append paged packed", "head_dim"),
    (dict(heads=5), "paged packed", "kv heads"), (dict(heads=-2), "paged packed", "kv heads"),
    (dict(window=-1), "paged packed", "window"), (dict(row_stride=HEADS * DIM - 1), "paged packed", "overlap"),
    (dict(row_stride=KV * DIM - 1), "append", "overlap"), (dict(row_stride=-1), "append paged packed", "overlap"),
    (dict(kv_stride=KV * DIM - 1), "packed", "overlap"), (dict(row_stride=1 << 20), "append paged packed", "out of range"),
    (dict(kv_stride=1 << 20), "packed", "out of range"),
])
def test_sizes_that_are_none(change, calls, text):
    for call in calls.split():
        c = getattr(Call(**change), call)
        if change == dict(dim=0) and call != "append":
            text = "head_dim" if call == "packed" else "out of range"
        refused(c(), text)


def test_heads_that_are_too_many():
    refused(Call(kv_heads=1 << 18, dim=128, pages=1, heads=1 << 18).paged(), "too large")
    big = buf(1 << 62, 1 << 20)
    refused(Call(kv_heads=1 << 18, dim=128, heads=1 << 18, q=big, out=buf(1 << 50, 1 << 63)).packed(), "too large")
    refused(Call(kv_heads=1 << 40, dim=128, heads=1 << 40).packed(), "out of range")
    refused(Call(kv_heads=1 << 28, dim=256, heads=1 << 28).packed(), "too large", OVERFLOW)
    refused(Call(kv_heads=1 << 28, dim=256).append(), "too large", OVERFLOW)
    refused(Call(rows=1 << 24, kv_heads=1, dim=1, heads=1 << 8, q=big, out=buf(1 << 50, 1 << 63)).packed(), "too large")


def test_what_is_missing():
    c, none = Call(), None
    b, L = c.b, lib()
    refused(L.accel_hip_batch_tables(b["counts"], b["lengths"], none, C.byref(c.batch), b["slots"], b["positions"],
                                     b["lengths_after"], b["state_after"]), "pool is missing")
    refused(L.accel_hip_batch_tables(b["counts"], b["lengths"], C.byref(c.pool), none, b["slots"], b["positions"],
                                     b["lengths_after"], b["state_after"]), "batch is missing")
    refused(L.accel_hip_release_pages(b["keep"], b["lengths"], none, C.byref(c.batch)), "pool is missing")
    refused(L.accel_hip_release_pages(b["keep"], b["lengths"], C.byref(c.pool), none), "batch is missing")
    refused(L.accel_hip_append_paged(b["k"], b["v"], none, b["slots"], 1, 0), "cache is missing")
    refused(L.accel_hip_attention_paged(b["q"], none, C.byref(c.batch), b["out"], 4, 0, 0), "cache is missing")
    refused(L.accel_hip_attention_paged(b["q"], C.byref(c.cache), none, b["out"], 4, 0, 0), "batch is missing")
    refused(L.accel_hip_attention_packed(b["q"], b["k"], b["v"], none, b["out"], 4, 2, 64, 0, 0, 0), "batch is missing")


def test_an_f16_cache_takes_half_the_bytes():
    """Its planes are checked by their own size and alignment."""
    size = PLACES["k_pages"][1] // 2
    for call in ("append", "paged"):
        refused(getattr(Call(type=CACHE_F16, k_pages=buf(size - 1, 13 * GIB)), call)(), "keys are out of range")
        refused(getattr(Call(type=CACHE_F16, v_pages=buf(size, 14 * GIB + 1)), call)(), "values are not aligned")
        # Enough, and 2-byte aligned: the next check refuses.
        refused(getattr(Call(type=CACHE_F16, k_pages=buf(size, 13 * GIB + 2), v_pages=buf(size, 13 * GIB + 2), window=-1), call)(),
                "overlap" if call == "append" else "window")


def test_the_slots_of_a_batch():
    """Where a batch has them, attention over pages checks them like its other parts; the other calls do not look."""
    at, size = PLACES["slots"]
    for slots, text in ((buf(size - 1, at * GIB), "slots are out of range"), (buf(size, at * GIB + 2), "slots are out of range"),
                        (buf(size, PLACES["out"][0] * GIB), "overlap"), (buf(size, PLACES["out"][0] * GIB + 4 - size), "overlap"),
                        (buf(size, PLACES["out"][0] * GIB + PLACES["out"][1] - 4), "overlap")):
        c = Call()
        c.batch.slots = slots
        refused(c.paged(), text)
        c = Call(window=-1)  # refused for that, behind the checks of the batch
        c.batch.slots = slots
        refused(c.packed(), "window")
    c = Call(window=-1)
    c.batch.slots = buf(size, at * GIB)
    refused(c.paged(), "window")
    c = Call(page=8)
    c.batch.slots = buf(1, at * GIB + 1)
    refused(c.tables(), "power of two")
    refused(c.release(), "power of two")


assert INVALID == 1
