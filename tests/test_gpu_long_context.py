"""Rotary positions, the 8-bit cache and attention over it, and sliding-window attention through the C-ABI,
against plain forms in 64 bits (long_context_helpers.py, which also says where each bound comes from)."""

from __future__ import annotations

import ctypes as C
import subprocess
import sys
import threading
from pathlib import Path

import numpy as np
import pytest

from accelep_amd.capi import Buffer, RopeScaling
from long_context_helpers import (NONE, Cache, append_call, assert_within, attend, attention_q8_call,
                                  attention_window_call, capi, check, dev, frequencies, lib, rotated)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    check(lib().accel_hip_init())
    yield


def say(*what):
    print(*what, flush=True)


# ---- rotary positions ----------------------------------------------------------------------------

@pytest.mark.parametrize("kind", range(5))
@pytest.mark.parametrize("rotary", [64, 128, 6])
def test_rope_frequencies(kind, rotary):
    s = RopeScaling(kind=kind, theta=1e5, factor=8.0, original_context=4096.0, fast=4.0 if kind == 4 else 32.0, slow=1.0)
    d, magnitude = dev(np.full(rotary // 2 + 1, 7.0)), C.c_float()
    check(lib().accel_hip_rope_frequencies(C.byref(s), rotary, d.buffer, C.byref(magnitude)))
    got = d.numpy()
    # pow and log of two libraries: a few ulp, times the logarithm of the base
    np.testing.assert_allclose(got[:-1], frequencies(kind, rotary, fast=s.fast), rtol=1e-13)
    assert got[-1] == 7.0
    assert magnitude.value == (np.float32(0.1 * np.log(8.0) + 1) if kind == capi.ROPE_SCALE_YARN else 1.0)


def rope_call(x, f, seq, heads, dim, rotary, layout, position=0, given=None, stride=0, magnitude=1.0, out=None):
    d = x if out is None else out
    g = dev(np.asarray(given, np.int32)) if given is not None else None
    fd = dev(f) if len(f) else None
    check(lib().accel_hip_rope_scaled(x.buffer, d.buffer, fd.buffer if fd else NONE, g.buffer if g else NONE, seq, heads,
                                      dim, stride, rotary, layout, position, magnitude))
    return d.numpy()


# Whole heads and parts, dims that take 16-byte loads and odd ones, one row to many, far positions.
@pytest.mark.parametrize("layout", [capi.ROPE_HALF, capi.ROPE_INTERLEAVED])
@pytest.mark.parametrize("seq,heads,dim,rotary,extra,position", [
    (1, 12, 64, 64, 0, 2047), (1, 1, 2, 2, 0, 0), (5, 3, 64, 32, 8, 100003), (3, 7, 100, 100, 3, 17), (9, 2, 80, 24, 4, 5),
    (33, 40, 128, 128, 1024, 131071), (2, 300, 96, 30, 1, 8), (4, 2, 33, 6, 0, 3), (3, 2, 256, 256, 0, (1 << 31) - 300),
    (1, 4, 64, 0, 0, 3)])
@pytest.mark.parametrize("in_place", [False, True])
def test_rope(layout, seq, heads, dim, rotary, extra, position, in_place):
    say("rope", layout, seq, heads, dim, rotary, extra, position, in_place)
    r = np.random.default_rng(seq + heads + dim + rotary)
    width = heads * dim + extra
    x = r.standard_normal((seq, width)).astype(np.float32)
    f = frequencies(capi.ROPE_SCALE_NONE, rotary)
    behind = np.full((seq, width), 5.0, np.float32)
    xd, out = dev(x), dev(behind)
    got = rope_call(xd, f, seq, heads, dim, rotary, layout, position, stride=width, magnitude=1.25, out=xd if in_place else out)
    want, bound = rotated(x[:, :heads * dim].reshape(seq, heads, dim), f, position + np.arange(seq), layout,
                          np.float64(np.float32(1.25)))
    assert_within(got[:, :heads * dim].reshape(seq, heads, dim), want, bound, floor=0)
    np.testing.assert_array_equal(got[:, heads * dim:], (x if in_place else behind)[:, heads * dim:])


@pytest.mark.parametrize("layout", [capi.ROPE_HALF, capi.ROPE_INTERLEAVED])
def test_rope_at_given_positions(layout):
    """Rows of several sequences; the largest given position, and one before the start."""
    r = np.random.default_rng(5)
    x = r.standard_normal((6, 4, 64)).astype(np.float32)
    given = np.array([0, 7, 7, 2 ** 31 - 1, 12345, -40], np.int32)
    f = frequencies(capi.ROPE_SCALE_YARN, 64)
    got = rope_call(dev(x), f, 6, 4, 64, 64, layout, position=1000, given=given, out=dev(np.zeros_like(x)))
    want, bound = rotated(x, f, 1000 + given.astype(np.int64), layout, 1.0)
    # 2^31 radians come out of one product in 64 bits, 2^31 * 2^-52 off at most
    assert_within(got, want, bound + 4 * 2.0 ** -21 * (np.abs(given.astype(np.float64)) > 2 ** 30)[:, None, None], floor=0)


def test_rope_from_memory_that_is_not_aligned_to_16_bytes():
    r = np.random.default_rng(6)
    host = r.standard_normal(3 * 128 + 1).astype(np.float32)
    d, f = dev(host), frequencies(capi.ROPE_SCALE_NONE, 64)
    fd = dev(f)
    at = Buffer(d.ptr + 4, 4 * 3 * 128, 0)
    check(lib().accel_hip_rope_scaled(at, at, fd.buffer, NONE, 3, 2, 64, 0, 64, 0, 11, 1.0))
    want, bound = rotated(host[1:].reshape(3, 2, 64), f, 11 + np.arange(3), 0, 1.0)
    got = d.numpy()
    assert got[0] == host[0]
    assert_within(got[1:].reshape(3, 2, 64), want, bound, floor=0)


@pytest.mark.parametrize("layout", [capi.ROPE_HALF, capi.ROPE_INTERLEAVED])
def test_rope_of_more_rows_than_a_grid_holds(layout):
    """2^23 rows and some: workgroups take several. The last rows are compared."""
    r = np.random.default_rng(7)
    rows = (1 << 23) + 1001
    x = np.tile(r.standard_normal((1001, 2)).astype(np.float32), (rows // 1001 + 1, 1))[:rows].reshape(rows, 1, 2)
    f = np.array([0.001])
    got = rope_call(dev(x), f, rows, 1, 2, 2, layout, out=dev(np.zeros_like(x)))
    for at in (slice(0, 50), slice((1 << 23) - 50, (1 << 23) + 50), slice(rows - 50, rows)):
        want, bound = rotated(x[at], f, np.arange(rows)[at], layout, 1.0)
        assert_within(got[at], want, bound, floor=0)


def test_append_of_more_blocks_than_a_grid_holds():
    """2^23 units and some, from inside a block: the launches meet at a block's border."""
    r = np.random.default_rng(15)
    kv, dim, block, position = 64, 1, 4, 2
    seq = (1 << 23) // (kv * 2) * block + 9
    cache = Cache(position + seq, kv, dim, block)
    first = [r.standard_normal((position, kv, dim)).astype(np.float32) for _ in "kv"]
    append_call(cache, *first, 0)
    cache.append(*first, 0)
    x = np.tile(r.standard_normal((1003, kv, dim)).astype(np.float32), (seq // 1003 + 1, 1, 1))[:seq]
    append_call(cache, x, -x, position)
    codes, scale = cache.on_device()
    whole = np.zeros((scale["k"].shape[0] * block, kv), np.float32)
    whole[:position], whole[position:position + seq] = first[0][..., 0], x[..., 0]
    need = (np.abs(whole.reshape(-1, block, kv).astype(np.float64)).max(axis=1) / 127).astype(np.float32)
    np.testing.assert_array_equal(scale["k"], need)
    by_row = np.repeat(need, block, axis=0)[position:position + seq].astype(np.float64)
    np.testing.assert_array_equal(codes["k"][position:, :, 0], np.rint(x[..., 0] / by_row))
    np.testing.assert_array_equal(codes["v"][position:, :, 0], np.rint(-x[..., 0] / np.repeat(scale["v"], block, axis=0)[position:position + seq]
                                                                       .astype(np.float64)))


def test_attention_of_nothing():
    L = lib()
    cache = Cache(16, 2, 64, 4)
    out = dev(np.full(64, 7.0, np.float32))
    for seq, heads in ((0, 4), (3, 0)):
        check(L.accel_hip_attention_q8(out.buffer if seq == 0 else NONE, C.byref(cache.handle), out.buffer, seq, 5, heads, 0, 0, 0))
        check(L.accel_hip_attention_window(NONE, cache.d_scale["k"].buffer if heads == 0 else NONE, NONE, NONE, 0, 0, heads, 2, 64, 0, 3, 1))
    check(L.accel_hip_append_cache_q8(NONE, NONE, C.byref(cache.handle), 0, 16, 0))
    check(L.accel_hip_read_cache_q8(C.byref(cache.handle), 16, 0, NONE, NONE))
    assert (out.numpy() == 7.0).all()


def test_rope_of_nothing():
    x = dev(np.zeros(64, np.float32))
    for seq, heads, dim in ((0, 2, 64), (3, 0, 64), (3, 2, 0)):
        check(lib().accel_hip_rope_scaled(x.buffer, x.buffer, NONE, NONE, seq, heads, dim, 0, 0, 0, 0, 1.0))


# ---- the 8-bit cache, written and read back ------------------------------------------------------

def assert_same_cache(cache):
    codes, scale = cache.on_device()
    for n in "kv":
        np.testing.assert_array_equal(scale[n], cache.scale[n])
        np.testing.assert_array_equal(codes[n], cache.codes[n])


def read_call(cache, first, count, k=True, v=True):
    shape = (count, *cache.shape[1:])
    out = [dev(np.full(shape, 9.0, np.float32)) if wanted else None for wanted in (k, v)]
    check(lib().accel_hip_read_cache_q8(C.byref(cache.handle), first, count, *(o.buffer if o else NONE for o in out)))
    return [o.numpy() if o else None for o in out]


# Rows arrive in parts that end inside blocks and at their borders, one by one, and many blocks at once; dims for
# 4-byte codes and odd ones; units that a wave holds, that a workgroup holds and that are read twice.
@pytest.mark.parametrize("kv_heads,dim,block,parts", [
    (3, 64, 64, [1, 1, 5, 57, 64, 65, 1]), (8, 128, 64, [100, 300]), (2, 128, 1, [1, 7, 130]), (1, 256, 256, [300, 1, 211]),
    (2, 100, 16, [3, 40, 1, 1]), (3, 33, 4, [1, 2, 3, 30]), (1, 1, 8, [1, 1, 20]), (2, 255, 128, [130, 70]),
    (5, 80, 32, [31, 1, 1, 31]), (1, 64, 256, [1] * 12)])
def test_append_and_read(kv_heads, dim, block, parts):
    say("append", kv_heads, dim, block, parts)
    r = np.random.default_rng(kv_heads * 1000 + dim + block)
    cache = Cache(sum(parts) + 3, kv_heads, dim, block)
    cache.fill(r, 0)
    for n in "kv":  # what lies behind is left as it is
        cache.codes[n][:] = 77
        cache.scale[n][:] = 3.5
    cache.upload()
    position = 0
    for seq in parts:
        k, v = (r.standard_normal((seq, kv_heads, dim)).astype(np.float32) * np.float32(1 + position % 7) for _ in "kv")
        append_call(cache, k, v, position)
        cache.append(k, v, position)
        position += seq
        assert_same_cache(cache)
    for first, count in ((0, position), (position // 2, 1), (position // 3, position - position // 3), (position, 0)):
        for n, got in zip("kv", read_call(cache, first, count)):
            np.testing.assert_array_equal(got, cache.values(n)[first:first + count])
    k_only = read_call(cache, 1, position - 1, v=False)[0]
    np.testing.assert_array_equal(k_only, cache.values("k")[1:position])


def test_append_again_at_an_earlier_position():
    """Rejected drafts are written over: the block keeps the scale it has where the rows before need it."""
    r = np.random.default_rng(3)
    cache = Cache(96, 2, 64, 32)
    for position, seq, gain in ((0, 40, 1.0), (37, 5, 4.0), (38, 3, 0.1), (32, 2, 0.01), (0, 1, 1.0), (64, 32, 1.0)):
        k, v = (gain * r.standard_normal((seq, 2, 64)) for _ in "kv")
        k, v = k.astype(np.float32), v.astype(np.float32)
        append_call(cache, k, v, position)
        cache.append(k, v, position)
        assert_same_cache(cache)


def test_append_of_rows_of_a_fused_projection():
    r = np.random.default_rng(4)
    rows = r.standard_normal((50, 6 * 64 + 2 * 2 * 64)).astype(np.float32)
    cache = Cache(64, 2, 64, 16)
    d = dev(rows)
    k, v = (Buffer(d.ptr + 4 * (6 * 64 + i * 128), rows.nbytes - 4 * (6 * 64 + i * 128), 0) for i in range(2))
    check(lib().accel_hip_append_cache_q8(k, v, C.byref(cache.handle), 50, 9, rows.shape[1]))
    cache.append(rows[:, 384:512].reshape(50, 2, 64), rows[:, 512:].reshape(50, 2, 64), 9)
    assert_same_cache(cache)


@pytest.mark.parametrize("gain", [1.0, 2.0 ** -120, 2.0 ** -140, 2.0 ** 120])
def test_codes_are_the_nearest_of_the_true_quotient(gain):
    """Values at and next to the border between two codes, at scales whose reciprocal is not finite too."""
    r = np.random.default_rng(8)
    dim, block = 256, 4
    # 127 * s as the largest makes the scale s (or its neighbour); (n + 1/2) s and its neighbours on both sides
    s = (1 + r.integers(0, 1 << 12, (64, 1, 1)) / 4096.0) * gain
    n = r.integers(-126, 127, (64, 1, dim)) + 0.5
    x = (n * s).astype(np.float32)
    x[:, :, 1::3] = np.nextafter(x[:, :, 1::3], np.float32(np.inf))
    x[:, :, 2::3] = np.nextafter(x[:, :, 2::3], np.float32(-np.inf))
    x[::block, :, 0] = (127 * s[::block, :, 0]).astype(np.float32)
    cache = Cache(64, 1, dim, block)
    append_call(cache, x, -x, 0)
    cache.append(x, -x, 0)
    assert_same_cache(cache)


@pytest.mark.parametrize("dim", [64, 63])
def test_codes_of_values_whose_scale_has_few_bits(dim):
    """Multiples of 2^-149 up to 2^14: the scale is one of few, a code may want 190 and is 127."""
    r = np.random.default_rng(31)
    cache = Cache(64, 3, dim, 4)
    top = np.float64(2.0) ** r.uniform(0, 14, (64, 3, 1)).round(2)
    top[:4] = 190
    top[4:8] = 63  # no scale at all
    k, v = ((np.rint(top * r.uniform(-1, 1, (64, 3, dim))) * 2.0 ** -149).astype(np.float32) for _ in "kv")
    k[0, :, 0] = 190 * 2.0 ** -149
    append_call(cache, k, v, 0)
    cache.append(k, v, 0)
    codes, scale = cache.on_device()
    for n in "kv":
        np.testing.assert_array_equal(scale[n], cache.scale[n])
        np.testing.assert_array_equal(codes[n], cache.codes[n])
    assert codes["k"][0, 0, 0] == 127 and (codes["k"][4:8] == 0).all()


def test_zeros_infinities_and_nans():
    cache = Cache(64, 2, 64, 16)
    r = np.random.default_rng(9)
    x = r.standard_normal((64, 2, 64)).astype(np.float32)
    x[:16, 0] = 0
    x[20, 1, 5] = np.inf
    x[40, 0, 63] = np.nan
    append_call(cache, x, x, 0)
    cache.append(x, x, 0)
    assert np.isnan(cache.scale["k"][1, 1]) and np.isnan(cache.scale["k"][2, 0]) and np.isnan(cache.scale["k"]).sum() == 2
    assert_same_cache(cache)
    for n, got in zip("kv", read_call(cache, 0, 64)):
        np.testing.assert_array_equal(got, cache.values(n))
    # zeros, then values in the same block; a NaN block stays one until its start is written again
    for position, seq in ((8, 4), (41, 3), (32, 2), (21, 3)):
        append_call(cache, x[:seq] + 1, x[:seq] - 1, position)
        cache.append(x[:seq] + 1, x[:seq] - 1, position)
        assert_same_cache(cache)


# ---- attention -----------------------------------------------------------------------------------

# (seq, position, heads, kv_heads, dim, block, window, sinks): one row and a few, whole row blocks and odd ones, one
# head a group to many; dims of whole 16 bytes and odd ones; windows of one key, that end inside blocks, that reach the
# start, that touch the first tokens; first tokens without a window, more of them than there are.
SHAPES = [
    (1, 0, 1, 1, 64, 64, 0, 0), (1, 63, 9, 3, 64, 64, 0, 0), (1, 64, 9, 3, 64, 64, 0, 0), (1, 2047, 9, 3, 64, 64, 0, 0),
    (1, 5000, 32, 8, 128, 16, 0, 0), (2, 700, 14, 2, 128, 32, 0, 0), (5, 1300, 8, 4, 128, 16, 300, 4),
    (7, 33, 4, 4, 80, 4, 0, 0), (3, 500, 6, 2, 100, 1, 0, 0), (4, 77, 3, 1, 33, 8, 20, 3), (1, 300, 2, 1, 256, 256, 0, 0),
    (2, 130, 2, 2, 1, 2, 0, 0), (1, 900, 5, 1, 64, 128, 1, 0), (1, 900, 5, 1, 64, 64, 1, 4), (3, 10, 2, 1, 64, 16, 50, 3),
    (1, 4000, 28, 4, 128, 64, 1000, 64), (1, 4000, 28, 4, 128, 64, 1000, 100), (2, 90, 4, 2, 64, 32, 0, 1000),
    (1, 200, 70, 1, 64, 64, 0, 0), (17, 0, 4, 2, 64, 64, 0, 0), (64, 0, 9, 3, 64, 64, 0, 0), (33, 200, 3, 1, 128, 32, 0, 0),
    (130, 61, 2, 2, 128, 64, 0, 0), (100, 1000, 4, 1, 64, 16, 64, 4), (65, 500, 6, 2, 96, 64, 1, 1),
    (40, 1000, 8, 2, 128, 1, 333, 70), (200, 3, 2, 1, 256, 128, 77, 0), (70, 300, 2, 1, 100, 4, 0, 0),
    (31, 129, 4, 2, 63, 32, 40, 8), (260, 0, 1, 1, 64, 256, 0, 0), (129, 640, 16, 4, 64, 64, 128, 128),
]
# And enough rows and keys for the kernels that bring tiles of keys through LDS: all dims and scale layouts, row blocks
# and key tiles whole and partial, a range in several parts, windows narrower than a tile and wider, rows that see
# nothing of a tile.
SHAPES += [
    (300, 0, 64, 8, 64, 64, 0, 0), (130, 1500, 64, 8, 128, 64, 0, 0), (97, 4001, 32, 4, 128, 128, 0, 0),
    (77, 3000, 40, 8, 80, 16, 0, 0), (65, 2500, 64, 4, 100, 64, 0, 0), (90, 2000, 48, 3, 33, 4, 0, 0),
    (64, 2100, 64, 16, 256, 32, 0, 0), (200, 1001, 64, 64, 64, 1, 0, 0), (513, 700, 56, 8, 128, 64, 300, 4),
    (1000, 37, 64, 8, 64, 32, 150, 70), (2100, 0, 64, 8, 128, 256, 33, 2), (400, 5000, 32, 1, 96, 2, 1000, 1000),
    (700, 300, 64, 2, 64, 64, 500, 0), (300, 2000, 24, 8, 255, 8, 900, 5), (600, 900, 32, 32, 128, 64, 1, 0),
    (17, 30000, 32, 2, 128, 64, 0, 0), (2500, 100, 64, 8, 64, 64, 16, 300), (150, 3000, 32, 8, 1, 64, 0, 0),
]
# Decode steps over long ranges, where a workgroup serves several key heads: four, three, two and one of them.
SHAPES += [(1, 70000, 8, 4, 128, 64, 0, 0), (1, 100000, 9, 3, 64, 32, 0, 0), (2, 150000, 4, 2, 64, 64, 0, 0),
           (1, 40000, 8, 4, 256, 16, 0, 0), (1, 60000, 10, 5, 80, 64, 59000, 4), (3, 90000, 4, 4, 100, 64, 0, 0)]
IDS = ["-".join(map(str, s)) for s in SHAPES]


def some_rows(seq):
    if seq <= 40:
        return np.arange(seq)
    return np.unique(np.r_[0:9, 15:18, 31:34, seq // 2, seq - 9:seq] if seq <= 260 else np.r_[0:3, 31:33, seq // 2, seq - 3:seq])


@pytest.mark.parametrize("seq,position,heads,kv_heads,dim,block,window,sinks", SHAPES, ids=IDS)
def test_attention_q8(seq, position, heads, kv_heads, dim, block, window, sinks):
    say("attention_q8", seq, position, heads, kv_heads, dim, block, window, sinks)
    r = np.random.default_rng(seq * 7 + position + dim + window)
    cache = Cache(position + seq + 5, kv_heads, dim, block)
    cache.fill(r, position + seq + 5)  # rows behind the last are not seen
    q = r.standard_normal((seq, heads, dim)).astype(np.float32)
    k, v = (cache.codes[n].astype(np.float64) * np.repeat(cache.scale[n].astype(np.float64), block, axis=0)[:len(cache.codes[n]), :, None]
            for n in "kv")
    got = attention_q8_call(q, cache, position, window, sinks)
    rows = some_rows(seq)
    want, bound = attend(q, k[:position + seq], v[:position + seq], position, window, sinks, rows, cache.value_scale(position + seq))
    assert_within(got[rows], want, bound)


@pytest.mark.parametrize("seq,position,heads,kv_heads,dim,block,window,sinks", SHAPES, ids=IDS)
def test_attention_window(seq, position, heads, kv_heads, dim, block, window, sinks):
    say("attention_window", seq, position, heads, kv_heads, dim, window, sinks)
    r = np.random.default_rng(seq * 5 + position + dim + window)
    rows = position + seq
    q, k, v = (r.standard_normal(s).astype(np.float32) for s in ((seq, heads, dim), (rows + 2, kv_heads, dim), (rows + 2, kv_heads, dim)))
    v *= np.exp(r.standard_normal((rows + 2, 1, 1))).astype(np.float32)
    k[rows:] = v[rows:] = np.nan  # rows behind the last are not read
    got = attention_window_call(q, k, v, position, window, sinks)
    some = some_rows(seq)
    want, bound = attend(q, k[:rows], v[:rows], position, window, sinks, some)
    assert_within(got[some], want, bound)


@pytest.mark.parametrize("seq,position", [(1, 777), (3, 500), (70, 300)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 5)])
def test_attention_of_rows_of_a_fused_projection(seq, position, window, sinks):
    """q inside wider rows, at an address that is not a multiple of 16 bytes."""
    r = np.random.default_rng(1)
    width = 4 * 64 + 67
    rows = r.standard_normal((seq, width)).astype(np.float32)
    d = dev(rows)
    q = rows[:, 33:33 + 256].reshape(seq, 4, 64)
    at = Buffer(d.ptr + 4 * 33, rows.nbytes - 4 * 33, 0)
    cache = Cache(position + seq, 2, 64, 32)
    cache.fill(r, position + seq)
    k, v = cache.values("k"), cache.values("v")
    out = dev(np.zeros((seq, 4, 64), np.float32))
    check(lib().accel_hip_attention_q8(at, C.byref(cache.handle), out.buffer, seq, position, 4, width, window, sinks))
    want, bound = attend(q, k, v, position, window, sinks)
    assert_within(out.numpy(), want, bound)
    kd, vd = dev(k), dev(v)
    check(lib().accel_hip_attention_window(at, kd.buffer, vd.buffer, out.buffer, seq, position, 4, 2, 64, width, window, sinks))
    assert_within(out.numpy(), want, bound)


@pytest.mark.parametrize("seq,position,window,sinks,copies", [
    (1, 400, 100, 4, 1), (5, 400, 100, 4, 1), (80, 400, 100, 4, 1), (200, 0, 33, 2, 1), (80, 400, 100, 4, 128), (200, 0, 33, 2, 128)])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf, 3e38])
def test_keys_that_a_row_does_not_see_do_not_reach_it(seq, position, window, sinks, copies, value):
    """One key and its value are not finite (or huge): the rows that see it may be anything, the others keep their
    results. Keys before the window and behind the first tokens, inside and at its border, and future ones."""
    r = np.random.default_rng(2)
    rows = position + seq
    q, k, v = (r.standard_normal(s).astype(np.float32) for s in ((seq, 4, 64), (rows, 2, 64), (rows, 2, 64)))
    for t in sorted({4, max(0, position - window), max(0, position - window + 1), position + seq // 2, rows - 1}):
        kk, vv = k.copy(), v.copy()
        kk[t, 0, 3] = vv[t, 0, 5] = value
        # `copies` of each query head: more rows, for the kernel of many of them
        got = attention_window_call(np.repeat(q, copies, axis=1), kk, vv, position, window, sinks)
        np.testing.assert_array_equal(got[:, 1::copies], got[:, ::copies]) if copies > 1 else None
        got = got[:, ::copies]
        p = position + np.arange(seq)
        blind = np.flatnonzero(~((t <= p) & ((t > p - window) | (t < sinks))))
        want, bound = attend(q, np.nan_to_num(kk, posinf=0, neginf=0), np.nan_to_num(vv, posinf=0, neginf=0), position,
                             window, sinks, blind)
        assert_within(got[blind], want, bound)
        others, bound = attend(q[:, 2:], k[:, 1:], v[:, 1:], position, window, sinks)
        assert_within(got[:, 2:], others, bound)  # the other key head
        if not np.isfinite(value):
            seen = np.setdiff1d(np.arange(seq), blind)
            assert not np.isfinite(got[seen, :2, 5]).any()


@pytest.mark.parametrize("seq,position,window,sinks,block,copies", [
    (1, 400, 100, 4, 16, 1), (6, 400, 100, 4, 32, 1), (80, 400, 100, 4, 8, 1), (200, 0, 33, 2, 64, 1), (90, 100, 0, 0, 16, 1),
    (80, 400, 100, 4, 8, 128), (200, 0, 33, 2, 64, 256), (90, 100, 0, 0, 16, 256), (200, 300, 64, 4, 32, 64)])
def test_blocks_that_a_row_does_not_see_do_not_reach_it(seq, position, window, sinks, block, copies):
    """A NaN scale makes a block's keys (or values) NaN: rows that see none of the block keep their results."""
    r = np.random.default_rng(4)
    rows = position + seq
    cache = Cache(rows, 2, 64, block)
    cache.fill(r, rows)
    q = r.standard_normal((seq, 4, 64)).astype(np.float32)
    clean = {n: cache.values(n) for n in "kv"}
    for plane in "kv":
        for b in sorted({1, max(0, position - window) // block, (position + seq // 2) // block, (rows - 1) // block}):
            kept = cache.scale[plane][b, 0]
            cache.scale[plane][b, 0] = np.nan
            cache.upload()
            got = attention_q8_call(np.repeat(q, copies, axis=1), cache, position, window, sinks)[:, ::copies]
            cache.scale[plane][b, 0] = kept
            p = position + np.arange(seq)[:, None]
            t = np.arange(b * block, min(rows, (b + 1) * block))[None, :]
            sees = (t <= p) & ((t > p - window) | (t < sinks) if window else True)
            blind = np.flatnonzero(~sees.any(axis=1))
            want, bound = attend(q, clean["k"], clean["v"], position, window, sinks, blind)
            assert_within(got[blind], want, bound)
            others, bound = attend(q[:, 2:], clean["k"][:, 1:], clean["v"][:, 1:], position, window, sinks)
            assert_within(got[:, 2:], others, bound)
            seen = np.flatnonzero(sees.any(axis=1))
            assert np.isnan(got[seen, :2]).all()


@pytest.mark.parametrize("seq,block", [(1, 16), (40, 16), (1, 64), (40, 64)])
@pytest.mark.parametrize("copies", [1, 128])
def test_attention_q8_over_scales_of_many_magnitudes(seq, block, copies):
    """Blocks whose scales lie apart by up to 2^16 in values, and queries whose rows do by 2^40: the weights' range."""
    r = np.random.default_rng(6)
    cache = Cache(600, 1, 64, block)
    cache.fill(r, 600)
    cache.scale["v"][:] = 2.0 ** r.integers(-16, 1, cache.scale["v"].shape)
    cache.upload()
    q = (r.standard_normal((seq, 3, 64)) * 2.0 ** np.array([-20, 0, 3])[None, :, None]).astype(np.float32)
    q[:, 1, 7] *= 1000
    position = 600 - seq
    want, bound = attend(q, cache.values("k"), cache.values("v"), position, 0, 0, None, cache.value_scale(600))
    assert_within(attention_q8_call(np.repeat(q, copies, axis=1), cache, position)[:, ::copies], want, bound)


@pytest.mark.parametrize("seq", [1, 40])
@pytest.mark.parametrize("copies", [1, 160])
@pytest.mark.parametrize("exponent", [-100, 100])
def test_attention_q8_of_very_small_and_large_values(seq, copies, exponent):
    r = np.random.default_rng(7)
    cache = Cache(300, 2, 64, 32)
    cache.fill(r, 300)
    cache.scale["v"] *= np.float32(2.0 ** exponent)
    cache.upload()
    q = r.standard_normal((seq, 2, 64)).astype(np.float32)
    want, bound = attend(q, cache.values("k"), cache.values("v").astype(np.float64), 300 - seq, 0, 0)
    assert_within(attention_q8_call(np.repeat(q, copies, axis=1), cache, 300 - seq)[:, ::copies], want, bound, floor=0)


@pytest.mark.parametrize("seq,copies", [(3, 1), (64, 64)])
@pytest.mark.parametrize("low,high", [(-3, 3), (-40, 40), (-100, 20), (0, 0)])
def test_attention_window_over_rows_of_many_magnitudes(seq, copies, low, high):
    """Key and value rows whose magnitudes lie apart by powers of two: common ones, and ones that need their own."""
    r = np.random.default_rng(17)
    rows = 900
    q, k, v = (r.standard_normal(s).astype(np.float32) for s in ((seq, 4, 64), (rows, 2, 64), (rows, 2, 64)))
    v *= (2.0 ** r.integers(low, high + 1, (rows, 2, 1))).astype(np.float32)
    k *= (2.0 ** np.minimum(r.integers(low, high + 1, (rows, 2, 1)), 2)).astype(np.float32)
    k[::7], v[::5] = 0, 0
    want, bound = attend(q, k, v, rows - seq, 0, 0)
    assert_within(attention_window_call(np.repeat(q, copies, axis=1), k, v, rows - seq)[:, ::copies], want, bound)


@pytest.mark.parametrize("copies", [1, 128])
def test_a_block_of_large_values_that_counts_for_little(copies):
    """One block's values lie 2^90 above the others' and its scores 2^7 below: its weight, 2^-120 and less, times its
    values is next to nothing, and the weights of the others keep their bits."""
    r = np.random.default_rng(18)
    cache = Cache(640, 1, 64, 64)
    cache.fill(r, 640)
    cache.codes["k"][:, 0, 0] = 64
    cache.codes["k"][192:256, 0, 0] = -64
    cache.scale["k"][:] = 1 / 64
    cache.scale["v"][3] *= np.float32(2.0 ** 90)
    cache.upload()
    q = r.standard_normal((24, 2, 64)).astype(np.float32) / 8
    q[:, :, 0] = 400  # scores of +-50 from this dim: weights e^-100
    want, bound = attend(q, cache.values("k"), cache.values("v"), 616, 0, 0, None, cache.value_scale(640))
    assert_within(attention_q8_call(np.repeat(q, copies, axis=1), cache, 616)[:, ::copies], want, bound)


@pytest.mark.parametrize("seq", [1, 24])
def test_attention_of_keys_that_all_score_the_same_and_of_one_that_wins(seq):
    """A query of zeros weighs every key alike; a key far above the others leaves their weights nothing."""
    r = np.random.default_rng(8)
    cache = Cache(500, 1, 64, 64)
    cache.fill(r, 500)
    q = np.zeros((seq, 2, 64), np.float32)
    q[:, 1] = 40 * cache.values("k")[3, 0] / np.abs(cache.values("k")[3, 0]).max()
    want, bound = attend(q, cache.values("k"), cache.values("v"), 500 - seq, 0, 0)
    assert_within(attention_q8_call(q, cache, 500 - seq), want, bound)
    got = attention_window_call(q, cache.values("k"), cache.values("v"), 500 - seq)
    assert_within(got, want, bound)


@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_a_query_row_that_is_not_finite_stays_alone(value):
    r = np.random.default_rng(9)
    cache = Cache(300, 1, 64, 64)
    cache.fill(r, 300)
    for seq, copies in ((2, 1), (40, 1), (40, 256)):
        q = r.standard_normal((seq, 2, 64)).astype(np.float32)
        q[1, 0, 9] = value
        clean = q.copy()
        clean[1, 0, 9] = 0
        want, bound = attend(clean, cache.values("k"), cache.values("v"), 300 - seq, 0, 0)
        many = np.repeat(q, copies, axis=1)
        for got in (attention_q8_call(many, cache, 300 - seq),
                    attention_window_call(many, cache.values("k"), cache.values("v"), 300 - seq)):
            got = got[:, ::copies]
            assert np.isnan(got[1, 0]).all()
            keep = np.ones((seq, 2), bool)
            keep[1, 0] = False
            assert_within(got[keep], want[keep], bound[keep])


def test_more_rows_than_the_grid_has_in_one_dimension():
    r = np.random.default_rng(10)
    cache = Cache(3, 1, 64, 1)
    cache.fill(r, 3)
    heads = 70000
    q = r.standard_normal((1, heads, 64)).astype(np.float32)
    some = np.r_[0:5, heads - 5:heads]
    want, bound = attend(q[:, some], cache.values("k"), cache.values("v"), 2, 0, 0)
    assert_within(attention_q8_call(q, cache, 2)[:, some], want, bound)
    assert_within(attention_window_call(q, cache.values("k"), cache.values("v"), 2)[:, some], want, bound)


def test_rows_past_the_reach_of_32_bit_offsets():
    """A cache of more than 2^32 codes, used at its end: written, read back and attended to."""
    kv_heads, dim, block, end = 8, 256, 64, (1 << 21) + 1000
    r = np.random.default_rng(11)
    L = lib()
    from accelep_amd.capi import CacheQ8
    from accelep_amd.device import DeviceArray
    codes = [DeviceArray((end, kv_heads, dim), np.int8) for _ in "kv"]
    scale = [DeviceArray((-(-end // block), kv_heads)) for _ in "kv"]
    handle = CacheQ8(*(x.buffer for x in codes + scale), end, kv_heads, dim, block)
    x = [r.standard_normal((200, kv_heads, dim)).astype(np.float32) for _ in "kv"]
    check(L.accel_hip_append_cache_q8(dev(x[0]).buffer, dev(x[1]).buffer, C.byref(handle), 200, end - 200, 0))
    out = [dev(np.zeros_like(x[0])) for _ in "kv"]
    check(L.accel_hip_read_cache_q8(C.byref(handle), end - 200, 200, out[0].buffer, out[1].buffer))
    k, v = (o.numpy() for o in out)
    for got, was in ((k, x[0]), (v, x[1])):
        assert np.abs(got - was).max() <= np.abs(was).max() / 127 * 0.51
    for seq in (1, 20):
        q = r.standard_normal((seq, 16, dim)).astype(np.float32)
        o = dev(np.zeros_like(q))
        check(L.accel_hip_attention_q8(dev(q).buffer, C.byref(handle), o.buffer, seq, end - seq, 16, 0, 100, 0))
        want, bound = attend(q, k[:, :], v[:, :], 200 - seq, 100, 0)
        assert_within(o.numpy(), want, bound)
    for a in codes + scale:
        a.free()
    check(L.accel_hip_trim())


# ---- as they are used together -------------------------------------------------------------------

def test_a_prompt_and_steps_over_the_cache():
    """A layer's attention over a growing 8-bit cache: prompt rows in two parts, then steps and one rejected draft,
    each rotated (YaRN, far positions), appended and attended to in a window with first tokens; against the same in
    64 bits. A value may come out one code apart where its rounded and its true rotation fall on two sides of a border,
    so the plain form codes the rotated rows that the device formed, after checking them."""
    r = np.random.default_rng(12)
    heads, kv, dim, rotary, block, window, sinks = 6, 2, 64, 48, 16, 100, 4
    f, magnitude = frequencies(capi.ROPE_SCALE_YARN, rotary), 0.1 * np.log(8.0) + 1
    cache = Cache(260, kv, dim, block)
    fd, L = dev(f), lib()
    width = (heads + 2 * kv) * dim
    for position, seq in ((0, 70), (70, 101), (171, 1), (172, 1), (173, 5), (175, 1), (176, 1)):
        say("layer", position, seq)
        rows = r.standard_normal((seq, width)).astype(np.float32)
        d = dev(rows)
        check(L.accel_hip_rope_scaled(d.buffer, d.buffer, fd.buffer, NONE, seq, heads + kv, dim, width, rotary,
                                      capi.ROPE_INTERLEAVED, position, magnitude))
        turned = d.numpy()
        want, bound = rotated(rows[:, :(heads + kv) * dim].reshape(seq, heads + kv, dim), f, position + np.arange(seq),
                              capi.ROPE_INTERLEAVED, np.float64(np.float32(magnitude)))
        assert_within(turned[:, :(heads + kv) * dim].reshape(want.shape), want, bound, floor=0)
        part = lambda at: Buffer(d.ptr + 4 * at * dim, rows.nbytes - 4 * at * dim, 0)  # noqa: E731
        check(L.accel_hip_append_cache_q8(part(heads), part(heads + kv), C.byref(cache.handle), seq, position, width))
        k, v = (turned[:, at * dim:(at + kv) * dim].reshape(seq, kv, dim) for at in (heads, heads + kv))
        cache.append(k, v, position)
        out = dev(np.zeros((seq, heads, dim), np.float32))
        check(L.accel_hip_attention_q8(d.buffer, C.byref(cache.handle), out.buffer, seq, position, heads, width, window, sinks))
        end = position + seq
        want, bound = attend(turned[:, :heads * dim].reshape(seq, heads, dim), cache.values("k")[:end],
                             cache.values("v")[:end], position, window, sinks)
        assert_within(out.numpy(), want, bound)
    assert_same_cache(cache)


def test_captured_and_replayed():
    """The calls of one step in a HIP graph, replayed with the eager calls between: the same bits each time."""
    r = np.random.default_rng(13)
    L = lib()
    heads, kv, dim, block = 8, 2, 128, 64
    for seq, position in ((1, 6000), (48, 2000), (700, 2000)):
        cache = Cache(position + seq, kv, dim, block)
        cache.fill(r, position + seq)
        x = r.standard_normal((seq, heads, dim)).astype(np.float32)
        k, v = (dev(r.standard_normal((seq, kv, dim)).astype(np.float32)) for _ in "kv")
        kf, vf = (dev(cache.values(n)) for n in "kv")
        xd, q, fd = dev(x), dev(np.zeros_like(x)), dev(frequencies(0, dim))
        outs = [dev(np.zeros_like(x)) for _ in range(2)]
        back = dev(np.zeros((seq, kv, dim), np.float32))

        def step():
            check(L.accel_hip_rope_scaled(xd.buffer, q.buffer, fd.buffer, NONE, seq, heads, dim, 0, dim, 0, position, 1.0))
            check(L.accel_hip_append_cache_q8(k.buffer, v.buffer, C.byref(cache.handle), seq, position, 0))
            check(L.accel_hip_attention_q8(q.buffer, C.byref(cache.handle), outs[0].buffer, seq, position, heads, 0, 0, 0))
            check(L.accel_hip_attention_window(q.buffer, kf.buffer, vf.buffer, outs[1].buffer, seq, position, heads, kv, dim, 0,
                                               1500, 4))
            check(L.accel_hip_read_cache_q8(C.byref(cache.handle), position, seq, back.buffer, NONE))

        def results():
            return [o.numpy() for o in (*outs, back)]

        step()
        eager = results()
        check(L.accel_hip_capture_begin())
        graph = C.c_void_p()
        try:
            step()
        finally:
            check(L.accel_hip_capture_end(C.byref(graph)))
        for replay in range(3):
            for o in (*outs, back, q):
                o.upload(np.full(o.shape, -1.0, np.float32))
            check(L.accel_hip_graph_launch(graph, 2))
            for got, want in zip(results(), eager):
                np.testing.assert_array_equal(got, want)
            step()
            for got, want in zip(results(), eager):
                np.testing.assert_array_equal(got, want)
        check(L.accel_hip_graph_destroy(graph))


def test_calls_from_two_threads_keep_their_sums_apart():
    """Both calls join key ranges in a second launch; the threads' launches meet on the one stream."""
    r = np.random.default_rng(17)
    L = lib()
    jobs = []
    for seq, heads, kv, dim, length in ((1, 32, 8, 128, 5000), (3, 9, 3, 64, 9000)):
        cache = Cache(length, kv, dim, 64)
        cache.fill(r, length)
        q = dev(r.standard_normal((seq, heads, dim)).astype(np.float32))
        kf, vf = (dev(cache.values(n)) for n in "kv")
        outs = [[dev(np.zeros(q.shape, np.float32)) for _ in range(2)] for _ in range(40)]

        def call(out, q=q, cache=cache, kf=kf, vf=vf, seq=seq, heads=heads, kv=kv, dim=dim, length=length):
            check(L.accel_hip_attention_q8(q.buffer, C.byref(cache.handle), out[0].buffer, seq, length - seq, heads, 0, 0, 0))
            check(L.accel_hip_attention_window(q.buffer, kf.buffer, vf.buffer, out[1].buffer, seq, length - seq, heads, kv, dim, 0,
                                               4000, 4))

        want = [dev(np.zeros(q.shape, np.float32)) for _ in range(2)]
        call(want)
        jobs.append((call, outs, [w.numpy() for w in want]))
    failures = []

    def run(call, outs):
        try:
            for out in outs:
                call(out)
        except BaseException as e:  # handed to the test's thread
            failures.append(e)

    threads = [threading.Thread(target=run, args=job[:2]) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures
    for _, outs, want in jobs:
        for out in outs:
            for got, w in zip(out, want):
                np.testing.assert_array_equal(got.numpy(), w)


FIRST_IN_A_CAPTURE = """
import ctypes as C, sys
sys.path[:0] = sys.argv[1:]
import numpy as np
from accelep_amd.capi import check, lib
from hip_helpers import dev
from long_context_helpers import Cache, assert_within, attend
L = lib()
check(L.accel_hip_init())
r = np.random.default_rng(19)
for seq in (1, 200):
    length, heads, kv, dim = 3000, 6, 2, 64
    cache = Cache(length, kv, dim, 64)
    cache.fill(r, length)
    x = r.standard_normal((seq, heads, dim)).astype(np.float32)
    k, v = cache.values("k"), cache.values("v")
    q, kf, vf = dev(x), dev(k), dev(v)
    outs = [dev(np.zeros_like(x)) for _ in range(2)]
    def step():
        check(L.accel_hip_attention_q8(q.buffer, C.byref(cache.handle), outs[0].buffer, seq, length - seq, heads, 0, 0, 0))
        check(L.accel_hip_attention_window(q.buffer, kf.buffer, vf.buffer, outs[1].buffer, seq, length - seq, heads, kv, dim, 0,
                                           2000, 4))
    check(L.accel_hip_capture_begin())
    graph = C.c_void_p()
    step()
    check(L.accel_hip_capture_end(C.byref(graph)))
    exact = [cache.codes[n].astype(np.float64) * np.repeat(cache.scale[n].astype(np.float64), 64, axis=0)[:length, :, None]
             for n in "kv"]
    wants = [attend(x, *exact, length - seq, 0, 0, value_scale=cache.value_scale(length)),
             attend(x, k, v, length - seq, 2000, 4)]
    for replay in range(3):
        for o in outs:
            o.upload(np.full(o.shape, -1.0, np.float32))
        check(L.accel_hip_graph_launch(graph, 1))
        for o, want in zip(outs, wants):
            assert_within(o.numpy(), *want)
    check(L.accel_hip_graph_destroy(graph))
    step()
    for o, want in zip(outs, wants):
        assert_within(o.numpy(), *want)
    print("held", seq, flush=True)
"""


def test_a_first_call_inside_a_capture():
    """Before any eager call there is no room for the parts of a key range: it stays whole."""
    here = Path(__file__).resolve().parent
    r = subprocess.run([sys.executable, "-c", FIRST_IN_A_CAPTURE, str(here), str(here.parent)], capture_output=True, text=True,
                       timeout=100)
    assert r.returncode == 0 and r.stdout.split() == ["held", "1", "held", "200"], r.stdout + r.stderr


def test_frequencies_are_refused_in_a_capture():
    L = lib()
    d, s, graph = dev(np.zeros(32)), RopeScaling(kind=0, theta=1e4), C.c_void_p()
    check(L.accel_hip_capture_begin())
    try:
        rc = L.accel_hip_rope_frequencies(C.byref(s), 64, d.buffer, None)
    finally:
        check(L.accel_hip_capture_end(C.byref(graph)))
        check(L.accel_hip_graph_destroy(graph))
    assert rc == 5
    assert not d.numpy().any()


def test_the_live_allocations_do_not_change():
    L = lib()
    r = np.random.default_rng(14)
    cache = Cache(300, 2, 64, 16)
    cache.fill(r, 300)
    q, out = dev(r.standard_normal((1, 4, 64)).astype(np.float32)), dev(np.zeros((1, 4, 64), np.float32))
    before = L.accel_hip_live_allocs()
    check(L.accel_hip_attention_q8(q.buffer, C.byref(cache.handle), out.buffer, 1, 299, 4, 0, 0, 0))
    assert L.accel_hip_live_allocs() == before
