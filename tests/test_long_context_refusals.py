"""What the long-context calls refuse, and with which status: decided on the host from the arguments
alone, so these tests need no GPU (the pointers are never read)."""

from __future__ import annotations

import ctypes as C

import pytest

from accelep_amd import capi
from accelep_amd.capi import Buffer, CacheQ8, RopeScaling, lib

INVALID, OVERFLOW = 1, 2
NONE = Buffer(None, 0, 0)


def buf(nbytes, at=1 << 20):
    return Buffer(at, nbytes, 0)


def cache(capacity=128, kv_heads=2, dim=64, block=32, **other):
    rows = max(capacity, 0) * max(kv_heads, 0) * max(dim, 0)
    scales = 4 * -(-max(capacity, 0) // max(block, 1)) * max(kv_heads, 0)
    fields = dict(k=buf(rows, 1 << 30), v=buf(rows, 2 << 30), k_scale=buf(scales, 3 << 30), v_scale=buf(scales, 4 << 30),
                  capacity=capacity, kv_heads=kv_heads, head_dim=dim, block=block)
    return CacheQ8(**{**fields, **other})


def refused(rc, text, status=INVALID):
    assert rc == status and text in lib().accel_hip_last_error().decode(), (rc, lib().accel_hip_last_error())


BAD_CACHES = [
    (dict(kv_heads=0), "shape"), (dict(dim=0), "shape"), (dict(capacity=-1), "shape"), (dict(dim=257), "head_dim"),
    (dict(block=0), "block"), (dict(block=24), "block"), (dict(block=512), "block"), (dict(block=-8), "block"),
    (dict(k=buf(128 * 2 * 64 - 1)), "keys"), (dict(v=NONE), "values"), (dict(k_scale=buf(31)), "key scales"),
    (dict(v_scale=buf(32, 2 + (1 << 20))), "not aligned"),
]


@pytest.mark.parametrize("change,text", BAD_CACHES, ids=[f"{sorted(c)[0]}-{i}" for i, (c, _) in enumerate(BAD_CACHES)])
def test_a_cache_of_no_form_is_refused_by_each_call(change, text):
    L, c = lib(), cache(**change)
    rows = buf(4 * 128 * 64 * 16)
    refused(L.accel_hip_append_cache_q8(rows, rows, C.byref(c), 1, 0, 0), text)
    refused(L.accel_hip_read_cache_q8(C.byref(c), 0, 1, rows, rows), text)
    refused(L.accel_hip_attention_q8(rows, C.byref(c), buf(1 << 20, 1 << 28), 1, 0, 4, 0, 0, 0), text)


def test_no_cache_is_refused():
    L, rows = lib(), buf(1 << 16)
    refused(L.accel_hip_append_cache_q8(rows, rows, None, 1, 0, 0), "missing")
    refused(L.accel_hip_read_cache_q8(None, 0, 1, rows, rows), "missing")
    refused(L.accel_hip_attention_q8(rows, None, rows, 1, 0, 4, 0, 0, 0), "missing")


def test_a_cache_too_large_to_count_is_an_overflow():
    L = lib()
    c = cache()
    c.capacity = 1 << 60
    refused(L.accel_hip_read_cache_q8(C.byref(c), 0, 1, buf(64), NONE), "too large", OVERFLOW)
    c = cache()
    c.kv_heads = 1 << 40
    refused(L.accel_hip_read_cache_q8(C.byref(c), 0, 1, buf(64), NONE), "too large", OVERFLOW)


def test_append_and_read_refuse_rows_out_of_range():
    L, c = lib(), cache()
    k, v = buf(4 * 4 * 128), buf(4 * 4 * 128, 1 << 28)
    call = lambda seq, position, stride=0, k=k, v=v: L.accel_hip_append_cache_q8(k, v, C.byref(c), seq, position, stride)  # noqa: E731
    refused(call(4, 125), "rows are out of range")
    refused(call(1, -1), "negative")
    refused(call(-1, 0), "negative")
    refused(call(2, (1 << 63) - 1), "too large", OVERFLOW)
    refused(call(5, 0), "keys are out of range")
    refused(call(4, 0, 127), "rows overlap")
    refused(call(4, 0, -128), "rows overlap")
    refused(call(4, 0, 129), "keys are out of range")  # the rows' spacing counts
    refused(call(4, 0, v=NONE), "values are out of range")
    refused(call(4, 0, k=buf(4 * 4 * 128, (1 << 20) + 2)), "not aligned")
    refused(call(4, 0, 1 << 62), "too large", OVERFLOW)
    read = lambda first, count, k=k, v=v: L.accel_hip_read_cache_q8(C.byref(c), first, count, k, v)  # noqa: E731
    refused(read(125, 4), "rows are out of range")
    refused(read(-1, 1), "negative")
    refused(read(0, -1), "negative")
    refused(read(0, 5), "key output")
    refused(read(0, 4, v=buf(4)), "value output")


def test_append_and_read_refuse_memory_that_is_written_twice():
    L = lib()
    k, v = buf(4 * 4 * 128), buf(4 * 4 * 128, 1 << 28)
    for name, other in (("v", buf(1 << 20, (1 << 30) + 100)), ("k_scale", buf(1 << 20, (1 << 30) + 4)),
                        ("v_scale", buf(1 << 20, 3 << 30)), ("v", buf(1 << 20, 1 << 28)), ("k_scale", buf(1 << 20, 1 << 20))):
        refused(L.accel_hip_append_cache_q8(k, v, C.byref(cache(**{name: other})), 4, 0, 0), "planes overlap")
    refused(L.accel_hip_append_cache_q8(buf(1 << 20, (2 << 30) + 4), v, C.byref(cache()), 4, 0, 0), "planes overlap")
    refused(L.accel_hip_read_cache_q8(C.byref(cache()), 0, 4, k, k), "outputs overlap")
    refused(L.accel_hip_read_cache_q8(C.byref(cache()), 0, 4, k, buf(1 << 20, (1 << 20) + 4 * 4 * 128 - 4)), "outputs overlap")


def test_attention_refuses_to_write_into_the_keys_and_values():
    L, c = lib(), cache()
    q = buf(4 * 3 * 4 * 64)
    for at in (1 << 30, (2 << 30) + 3 * 128 - 4):
        refused(L.accel_hip_attention_q8(q, C.byref(c), buf(1 << 20, at), 3, 0, 4, 0, 0, 0), "overlaps the cache")
    k, v = buf(4 * 128 * 2 * 64, 1 << 30), buf(4 * 128 * 2 * 64, 2 << 30)
    for at in (1 << 30, (2 << 30) + 4 * 3 * 128 - 4):
        refused(L.accel_hip_attention_window(q, k, v, buf(1 << 20, at), 3, 0, 4, 2, 64, 0, 0, 0), "overlaps the cache")


def test_attention_refuses_key_rows_past_its_offsets():
    L, wide = lib(), (1 << 17) + 1  # heads of 128: 2^24 + 128
    room, out = buf(1 << 40), buf(1 << 40, 1 << 50)
    c = cache(1, wide, 128, 1, **{n: buf(1 << 40, (i + 2) << 50) for i, n in enumerate(("k", "v", "k_scale", "v_scale"))})
    refused(L.accel_hip_attention_q8(room, C.byref(c), out, 1, 0, wide, 0, 0, 0), "too large")
    refused(L.accel_hip_attention_window(room, c.k, c.v, out, 1, 0, wide, wide, 128, 0, 0, 0), "too large")


def test_attention_refuses_what_does_not_fit():
    L, c = lib(), cache()
    q, out = buf(4 * 3 * 4 * 64), buf(4 * 3 * 4 * 64, 1 << 28)

    def q8(q=q, out=out, seq=3, position=0, heads=4, stride=0, window=0, sinks=0):
        return L.accel_hip_attention_q8(q, C.byref(c), out, seq, position, heads, stride, window, sinks)

    k, v = buf(4 * 128 * 2 * 64, 1 << 30), buf(4 * 128 * 2 * 64, 2 << 30)

    def window(q=q, out=out, seq=3, position=0, heads=4, stride=0, window=0, sinks=0, k=k, v=v, kv_heads=2, dim=64):
        return L.accel_hip_attention_window(q, k, v, out, seq, position, heads, kv_heads, dim, stride, window, sinks)

    for call in (q8, window):
        refused(call(heads=3), "kv heads")
        refused(call(heads=-2), "negative")
        refused(call(window=-1), "window")
        refused(call(window=4, sinks=-1), "window")
        refused(call(position=-1), "negative")
        refused(call(seq=-1), "negative")
        refused(call(q=buf(4 * 3 * 4 * 64 - 4)), "query is out of range")
        refused(call(out=buf(4 * 3 * 4 * 64 - 4, 1 << 28)), "output is out of range")
        refused(call(stride=255), "query rows overlap")
        refused(call(stride=257), "query is out of range")
        refused(call(q=buf(1 << 20, (1 << 20) + 1)), "not aligned")
        refused(call(out=q), "overlaps the query")
        refused(call(out=buf(1 << 20, (1 << 20) + 4 * 3 * 4 * 64 - 4)), "overlaps the query")
        refused(call(seq=2, position=(1 << 63) - 2), "too large", OVERFLOW)
        refused(call(seq=1, position=(1 << 31) - 1), "too large")
    refused(q8(position=126), "rows are out of range")
    refused(window(position=126), "key is out of range")
    refused(window(v=NONE), "value is out of range")
    refused(window(kv_heads=0), "kv heads")
    refused(window(dim=257, q=buf(1 << 20)), "head_dim")
    refused(window(dim=-64), "negative")
    refused(window(k=buf(1 << 20, (1 << 30) + 2)), "not aligned")


def test_rope_refuses_what_does_not_fit():
    L = lib()
    x, out, f = buf(4 * 3 * 128), buf(4 * 3 * 128, 1 << 28), buf(8 * 32, 1 << 29)

    def rope(x=x, out=out, f=f, positions=NONE, seq=3, heads=2, dim=64, stride=0, rotary=64, layout=0, position=0):
        return L.accel_hip_rope_scaled(x, out, f, positions, seq, heads, dim, stride, rotary, layout, position, 1.0)

    refused(rope(seq=-1), "negative")
    refused(rope(heads=-1), "negative")
    refused(rope(dim=-1), "negative")
    refused(rope(dim=258), "head_dim")
    refused(rope(rotary=63), "rotary_dim")
    refused(rope(rotary=66), "rotary_dim")
    refused(rope(rotary=-2), "rotary_dim")
    refused(rope(layout=2), "layout")
    refused(rope(layout=-1), "layout")
    refused(rope(position=-1), "negative")
    refused(rope(position=1 << 31), "position")
    refused(rope(seq=4), "states are out of range")
    refused(rope(out=buf(4 * 3 * 128 - 4, 1 << 28)), "output is out of range")
    refused(rope(stride=127), "rows overlap")
    refused(rope(stride=129), "states are out of range")
    refused(rope(out=buf(1 << 20, (1 << 20) + 4)), "overlaps")
    refused(rope(x=buf(1 << 20, (1 << 20) + 3)), "not aligned")
    refused(rope(f=buf(8 * 31, 1 << 29)), "frequencies are out of range")
    refused(rope(f=buf(8 * 32, (1 << 29) + 4)), "not aligned")
    refused(rope(positions=buf(8, 1 << 27)), "positions are out of range")
    refused(rope(positions=buf(12, (1 << 27) + 2)), "not aligned")


@pytest.mark.parametrize("rotary,change,text", [
    (64, dict(kind=5), "unknown"), (64, dict(kind=-1), "unknown"), (64, dict(theta=0.0), "theta"),
    (64, dict(theta=float("nan")), "theta"), (64, dict(theta=float("inf")), "theta"), (64, dict(factor=0.0), "factor"),
    (64, dict(factor=float("nan")), "factor"), (64, dict(fast=1.0), "borders"), (64, dict(slow=0.0), "borders"),
    (64, dict(original_context=0.0), "borders"), (64, dict(theta=1.0), "theta"), (2, dict(kind=2), "4 at least"),
    (63, {}, "rotary_dim"), (-2, {}, "rotary_dim"), (258, {}, "rotary_dim")])
def test_rope_frequencies_refuse_what_they_cannot_scale(rotary, change, text):
    fields = dict(kind=capi.ROPE_SCALE_YARN, theta=1e5, factor=8.0, original_context=4096.0, fast=32.0, slow=1.0)
    refused(lib().accel_hip_rope_frequencies(C.byref(RopeScaling(**{**fields, **change})), rotary, buf(8 * 129), None), text)


def test_rope_frequencies_refuse_no_scaling_and_no_room():
    s = RopeScaling(kind=0, theta=1e4)
    refused(lib().accel_hip_rope_frequencies(None, 64, buf(256), None), "missing")
    refused(lib().accel_hip_rope_frequencies(C.byref(s), 64, buf(255), None), "out of range")
    refused(lib().accel_hip_rope_frequencies(C.byref(s), 64, buf(256, (1 << 20) + 4), None), "not aligned")
