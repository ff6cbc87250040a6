"""The 8-bit cache after rows that were appended and then written over (a rejected draft)."""

from __future__ import annotations

import numpy as np
import pytest

from long_context_helpers import Cache, append_call, check, lib

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    check(lib().accel_hip_init())
    yield


def test_a_block_keeps_its_scale_over_dropped_rows_until_it_is_written_from_its_start():
    cache = Cache(64, 1, 64, 16)

    def append(value, seq, position):
        x = np.full((seq, 1, 64), value, np.float32)
        append_call(cache, x, -x, position)
        codes, scale = cache.on_device()
        np.testing.assert_array_equal(codes["v"], -codes["k"])
        return codes["k"][..., 0].ravel(), scale["k"].ravel()

    one, large = np.float32(1) / np.float32(127), np.float32(127 * 8) / np.float32(127)
    append(1.0, 20, 0)
    codes, scale = append(127 * 8.0, 15, 20)  # a draft of large values, over the second block's end into the third
    assert list(scale[:3]) == [one, large, large] and (codes[:16] == 127).all() and (codes[16:20] == 0).all()
    codes, scale = append(1.0, 15, 20)  # dropped: other rows in its place
    assert list(scale[:3]) == [one, large, one]  # the second block has rows before 20 and keeps its scale
    assert (codes[20:32] == 0).all() and (codes[32:35] == 127).all()
    codes, scale = append(1.0, 4, 16)  # written from its start
    assert list(scale[:3]) == [one, one, one] and (codes[16:20] == 127).all()
