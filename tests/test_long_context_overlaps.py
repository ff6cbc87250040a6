"""Outputs of the long-context calls over memory that the same call reads: refused on the host, so these tests need
no GPU (the pointers are never read)."""

from __future__ import annotations

import ctypes as C

import pytest

from accelep_amd.capi import lib
from test_long_context_refusals import NONE, buf, cache, refused

# cache(): 128 rows of 2 heads of 64 in blocks of 32; k, v, k_scale and v_scale lie at 1, 2, 3 and 4 GiB.
GIB = 1 << 30


@pytest.mark.parametrize("plane", [3, 4])
@pytest.mark.parametrize("rows,used", [(3, 1), (33, 2), (128, 4)])
def test_attention_refuses_to_write_into_the_scales(plane, rows, used):
    """The scales of the blocks that the call reads: `used` blocks of 2 heads."""
    L, q = lib(), buf(1 << 20)
    out_bytes = 4 * 1 * 4 * 64
    for at in (0, 4 * (2 * used - 1), 4 - out_bytes):
        refused(L.accel_hip_attention_q8(q, C.byref(cache()), buf(out_bytes, plane * GIB + at), 1, rows - 1, 4, 0, 0, 0),
                "overlaps the cache")


@pytest.mark.parametrize("first,count", [(0, 4), (30, 5), (124, 4)])
def test_a_read_refuses_to_write_into_what_it_reads(first, count):
    """The codes and scales of the rows that are read, for either output, alone and together; a plane that is left out
    is not read."""
    L, c = lib(), cache()
    bytes_out, code_row, blocks = 4 * count * 128, 128, (first // 32, (first + count - 1) // 32 + 1)
    clear = buf(bytes_out)
    for plane in "kv":
        codes, scales = (1, 3) if plane == "k" else (2, 4)
        for begin, size in ((codes * GIB + first * code_row, count * code_row),
                            (scales * GIB + 8 * blocks[0], 8 * (blocks[1] - blocks[0]))):
            for at in (begin, begin + size - 4, begin + 4 - bytes_out):
                out = buf(bytes_out, at)
                for k_out, v_out in ((out, clear), (clear, out), (out, NONE) if plane == "k" else (NONE, out)):
                    refused(L.accel_hip_read_cache_q8(C.byref(c), first, count, k_out, v_out), "overlap the cache")


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("stride", [0, 160])
def test_rope_refuses_to_write_into_its_frequencies_and_positions(in_place, stride):
    """3 rows of 2 heads of 64; 32 frequencies of 8 bytes and 3 positions of 4."""
    L, out = lib(), buf(1 << 20, GIB)
    x = out if in_place else buf(1 << 20, 2 * GIB)
    row, apart = 4 * 128, 4 * (stride or 128)
    f, p = buf(256, 3 * GIB), buf(12, 4 * GIB)

    def rope(f=f, p=p, rotary=64):
        return L.accel_hip_rope_scaled(x, out, f, p, 3, 2, 64, stride, rotary, 0, 0, 1.0)

    for at in (0, 8, row - 8, apart, 2 * apart + row - 8, 8 - 256, apart + 8 - 256):
        refused(rope(f=buf(256, GIB + at)), "overlaps the frequencies")
    for at in (0, 4, row - 4, 2 * apart + row - 4, 4 - 12, 2 * apart + 4 - 12):
        refused(rope(p=buf(12, GIB + at)), "overlaps the positions")
