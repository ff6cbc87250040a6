"""Tables of a batch's step, pages taken back and rows put into pages, through the C-ABI, against plain forms on
the host. Whole numbers have to be equal; a row in a page is its values rounded to the cache's type once."""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from accelep_amd import capi
from accelep_amd.capi import Batch, Buffer, CachePaged, PagePool, check, lib
from batch_helpers import TYPES, dev, ints, pool_of, released, tables

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    check(lib().accel_hip_init())
    yield


def say(*what):
    print(*what, flush=True)


class Step:
    """What one call reads and writes, on the host and on the device."""

    def __init__(self, rng, counts, lengths, page, rows, width, free, in_place=False):
        self.counts, self.lengths, self.page, self.rows = np.asarray(counts, np.int32), np.asarray(lengths, np.int32), page, rows
        requests = len(counts)
        have = [min(-(-max(int(n), 0) // page), width) for n in lengths]
        self.pages = sum(have) + free
        order = rng.permutation(self.pages).astype(np.int32)
        self.table = np.full((requests, width), -7, np.int32)
        for r, n in enumerate(have):
            self.table[r, :n] = order[sum(have[:r]):sum(have[:r]) + n]
        self.stack = np.full(max(self.pages, 1), -9, np.int32)
        self.stack[:free] = order[sum(have):]
        self.left = free
        self.d = {"counts": ints(self.counts), "lengths": ints(self.lengths), "table": ints(self.table),
                  "stack": ints(self.stack), "state": ints([free, 99])}
        for name, n in (("starts", requests + 1), ("seen", requests), ("slots", rows), ("positions", rows)):
            self.d[name] = ints(np.full(n, -55))
        self.d["lengths_after"] = self.d["lengths"] if in_place else ints(np.full(requests, -55))
        self.d["state_after"] = self.d["state"] if in_place else ints([-55, -55])
        b = {n: x.buffer for n, x in self.d.items()}
        self.pool = PagePool(b["stack"], b["state"], self.pages, page)
        self.batch = Batch(b["seen"], b["starts"], b["table"], requests, rows, width, 0)

    def call(self):
        b = {n: x.buffer for n, x in self.d.items()}
        check(lib().accel_hip_batch_tables(b["counts"], b["lengths"], C.byref(self.pool), C.byref(self.batch), b["slots"],
                                           b["positions"], b["lengths_after"], b["state_after"]))

    def want(self):
        return tables(self.counts, self.lengths, self.table, self.stack, self.left, self.rows, self.page, self.pages)

    def compare(self):
        for name, want in self.want().items():
            np.testing.assert_array_equal(self.d[name].numpy().ravel(), np.asarray(want).ravel(), err_msg=name)
        np.testing.assert_array_equal(self.d["stack"].numpy(), self.stack)


# requests, counts (a callable of rng), lengths, page, rows that are padding, width, free pages
def _some(rng, n, low, high):
    return rng.integers(low, high + 1, n)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("requests,count,length,page,pad", [
    (1, (1, 1), (0, 0), 16, 0), (1, (1, 1), (15, 16), 16, 3), (64, (1, 1), (0, 4000), 16, 0), (64, (0, 3), (0, 40), 32, 5),
    (7, (300, 900), (0, 100), 64, 1), (1000, (1, 2), (0, 300), 16, 40), (1025, (0, 1), (0, 64), 256, 0),
    (2049, (0, 2), (0, 40), 16, 9), (40, (100, 400), (0, 500), 16, 0), (9000, (0, 2), (0, 33), 16, 77), (3, (0, 0), (0, 9), 16, 4)])
def test_tables(requests, count, length, page, pad, in_place):
    say("tables", requests, count, length, page, pad, in_place)
    rng = np.random.default_rng(requests + page)
    counts, lengths = _some(rng, requests, *count), _some(rng, requests, *length)
    fresh = sum(-(-(a + b) // page) + -(-a // page) * -1 for a, b in zip(lengths.tolist(), counts.tolist()))
    s = Step(rng, counts, lengths, page, int(counts.sum()) + pad, int((lengths + counts).max() + page - 1) // page + 1,
             fresh + 5, in_place)
    s.call()
    s.compare()


def test_requests_that_get_no_page():
    """Too few free pages for the third and those behind it that need one; the others go on. A request that its table
    row is too short for takes nothing from the others."""
    rng = np.random.default_rng(3)
    counts, lengths = [20, 40, 33, 1, 1, 2, 500, 0], [0, 8, 0, 5, 16, 30, 3, 12]
    for free in range(0, 9):
        s = Step(rng, counts, lengths, 16, 620, 8, free)
        s.call()
        s.compare()


def test_rows_past_the_batch_do_not_count():
    rng = np.random.default_rng(4)
    for rows in (0, 1, 19, 20, 21, 59, 60):
        s = Step(rng, [20, 40, 5, -3, 2 ** 31 - 1], [0, 8, 0, 5, 4], 16, rows, 9, 12)
        s.call()
        s.compare()


def test_lengths_and_state_out_of_range():
    """Lengths below 0 count as 0, one past its table row gets nothing, a stack's count is kept to its size."""
    rng = np.random.default_rng(5)
    for left in (-5, 3, 1000, 2 ** 31 - 1):
        s = Step(rng, [3, 2, 1, 1], [-4, 2 ** 31 - 1, 16 * 5, 15], 16, 10, 5, 6)
        s.left = left
        s.d["state"].upload(np.array([left, 0], np.int32))
        s.stack[:] = np.arange(len(s.stack))
        s.d["stack"].upload(s.stack)
        s.call()
        got = {n: s.d[n].numpy() for n in ("starts", "seen", "slots", "lengths_after", "state_after")}
        left_now = min(max(left, 0), s.pages)
        served = left_now >= 1
        assert got["starts"].tolist() == [0, 3, 5, 6, 7] and got["seen"].tolist() == [0, 2 ** 31 - 1, 80, 15]
        assert got["lengths_after"].tolist() == [3 if served else 0, 2 ** 31 - 1, 80, 16]
        assert got["state_after"].tolist() == [left_now - served, 2 + (not served)]
        first = s.stack[left_now - 1] * 16 if served else 0
        assert got["slots"].tolist() == [*([first, first + 1, first + 2] if served else [-1] * 3), -1, -1, -1,
                                         s.table[3, 0] * 16 + 15, -1, -1, -1]


def test_pages_that_are_none_give_no_slot():
    rng = np.random.default_rng(6)
    s = Step(rng, [1, 1, 1], [3, 3, 16], 16, 3, 4, 2)
    s.table[:, 0] = [-1, s.pages, 0]
    s.d["table"].upload(s.table)
    s.stack[1] = 2 ** 31 - 1
    s.d["stack"].upload(s.stack)
    s.call()
    assert s.d["slots"].numpy().tolist() == [-1, -1, -1] and s.d["positions"].numpy().tolist() == [3, 3, 16]


def test_no_requests():
    rng = np.random.default_rng(7)
    for rows in (0, 5, 5000):
        s = Step(rng, [], [], 16, rows, 0, 4)
        s.call()
        s.compare()


@pytest.mark.parametrize("requests,chunk", [(5, 1), (50, 140)])
def test_a_captured_step_goes_on_by_itself(requests, chunk):
    """Lengths and the pool's state in place: each replay is the next step. Both forms of the call."""
    rng = np.random.default_rng(8)
    counts, lengths = rng.integers(1, chunk + 1, requests), rng.integers(0, 50, requests)
    s = Step(rng, counts, lengths, 16, int(counts.sum()) + 2, 80, 6 * int(counts.sum() // 16 + requests), True)
    s.call()  # also grows the scratch
    L, graph = lib(), C.c_void_p()
    check(L.accel_hip_capture_begin())
    s.call()
    check(L.accel_hip_capture_end(C.byref(graph)))
    try:
        for i in range(5):
            want = s.want()
            got = {n: s.d[n].numpy() for n in want}
            for name in want:
                np.testing.assert_array_equal(got[name].ravel(), np.asarray(want[name]).ravel(), err_msg=f"{name} {i}")
            s.lengths, s.table, s.left = np.asarray(want["lengths_after"], np.int32), want["table"], want["state_after"][0]
            check(L.accel_hip_graph_launch(graph, 1))
    finally:
        check(L.accel_hip_graph_destroy(graph))


# ---- pages taken back ----------------------------------------------------------------------------

@pytest.mark.parametrize("requests,length,page,width", [(1, 100, 16, 7), (3, 0, 16, 2), (64, 3000, 16, 190), (1500, 40, 32, 3),
                                                        (5, 20000, 64, 330)])
def test_release(requests, length, page, width):
    rng = np.random.default_rng(requests)
    lengths = rng.integers(0, length + 1, requests).astype(np.int32)
    keep = np.where(rng.random(requests) < 0.5, rng.integers(-2, length + 1, requests), lengths).astype(np.int32)
    have = -(-lengths // page)
    pages = int(have.sum()) + 9
    order = rng.permutation(pages).astype(np.int32)
    table = np.full((requests, width), -1, np.int32)
    for r in range(requests):
        table[r, :have[r]] = order[have[:r].sum():have[:r].sum() + have[r]]
    if requests > 1:
        table[requests // 2, 0] = pages + 4  # no page
    stack = np.full(pages, -9, np.int32)
    stack[:9] = order[-9:]
    want = released(keep, lengths, table, stack, 9, page, pages)
    pool, held = pool_of(stack, 9, page)
    held[1].upload(np.array([9, 5], np.int32))
    d = ints(keep), ints(lengths), ints(table)
    batch = Batch(capi.Buffer(None, 0, 0), capi.Buffer(None, 0, 0), d[2].buffer, requests, 0, width, 0)
    check(lib().accel_hip_release_pages(d[0].buffer, d[1].buffer, C.byref(pool), C.byref(batch)))
    for got, w in zip((d[1].numpy(), d[2].numpy(), held[0].numpy()), want):
        np.testing.assert_array_equal(got, w)
    assert held[1].numpy().tolist() == [want[3], 5]


def test_release_onto_a_full_stack_stays_inside_it():
    """More pages than there are (a page entered twice): the stack ends where it ends."""
    table = np.array([[0, 1, 1, 2], [2, 3, 0, 1]], np.int32)
    pool, held = pool_of([3, 2, -9, -9], 2, 16)
    d = ints([0, 0]), ints([64, 64]), ints(table)
    batch = Batch(capi.Buffer(None, 0, 0), capi.Buffer(None, 0, 0), d[2].buffer, 2, 0, 4, 0)
    check(lib().accel_hip_release_pages(d[0].buffer, d[1].buffer, C.byref(pool), C.byref(batch)))
    assert held[0].numpy().tolist() == [3, 2, 0, 1] and held[1].numpy()[0] == 4
    assert (d[2].numpy() == -1).all() and d[1].numpy().tolist() == [0, 0]


# ---- rows into pages -----------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("rows,kv_heads,dim,page,extra,shift", [
    (1, 3, 64, 16, 0, 0), (16, 8, 128, 64, 8, 0), (5, 1, 1, 16, 0, 0), (33, 2, 100, 32, 3, 0), (9, 3, 33, 16, 1, 0),
    (257, 2, 80, 256, 0, 0), (4, 1, 256, 16, 0, 1), (700, 8, 128, 16, 0, 0)])
def test_append(kind, rows, kv_heads, dim, page, extra, shift):
    """Whole rows and slices of wider ones, dims that fit 16-byte loads and others, memory that is not aligned to
    them (shift), slots outside the cache on both sides."""
    say("append", kind, rows, kv_heads, dim, page, extra, shift)
    rng = np.random.default_rng(rows + dim)
    pages, width, stride = 2 * rows // page + 2, kv_heads * dim, kv_heads * dim + extra
    slots = rng.permutation(pages * page)[:rows].astype(np.int32)
    slots[1::5] = -1
    slots[2::7] = pages * page
    x = {n: (rng.standard_normal(rows * stride + shift) * 3).astype(np.float32) for n in "kv"}
    x["k"][shift] = 1e30  # past the largest f16
    x["v"][shift] = 65519.0  # the largest that is not
    planes = {n: np.full(pages * page * width, 7, TYPES[kind]) for n in "kv"}
    d, src, sd = {n: dev(planes[n]) for n in "kv"}, {n: dev(x[n]) for n in "kv"}, ints(slots)
    cache = CachePaged(d["k"].buffer, d["v"].buffer, capi.CACHE_F16 if kind == "f16" else capi.CACHE_F32, pages, page, kv_heads, dim)
    at = [Buffer(src[n].at(shift), 4 * (rows * stride), 0) for n in "kv"]
    check(lib().accel_hip_append_paged(at[0], at[1], C.byref(cache), sd.buffer, rows, stride if extra else 0))
    for n in "kv":
        want = planes[n].reshape(-1, width)
        with np.errstate(over="ignore"):
            for i, s in enumerate(slots):
                if 0 <= s < pages * page:
                    want[s] = x[n][shift + i * stride:shift + i * stride + width].astype(TYPES[kind])
        np.testing.assert_array_equal(d[n].numpy().reshape(-1, width), want, err_msg=n)


def test_append_of_no_rows():
    d = dev(np.full(2 * 16 * 8, 7, np.float32))
    half = Buffer(d.ptr, 4 * 128, 0), Buffer(d.ptr + 4 * 128, 4 * 128, 0)
    cache = CachePaged(half[0], half[1], capi.CACHE_F32, 1, 16, 1, 8)
    none = Buffer(None, 0, 0)
    check(lib().accel_hip_append_paged(none, none, C.byref(cache), none, 0, 0))
    assert (d.numpy() == 7).all()
