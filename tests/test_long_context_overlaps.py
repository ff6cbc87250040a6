"""Outputs of the long-context calls over memory that the same call reads: refused on the host, so these tests need
no GPU (the pointers are never read)."""

from __future__ import annotations

import ctypes as C

import pytest

from accelep_amd.capi import lib
from test_long_context_refusals import buf, cache, refused

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
