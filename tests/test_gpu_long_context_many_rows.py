"""Attention over the 8-bit cache with enough rows for the kernel that brings tiles of keys through LDS: value scales
far apart, small and large, with a scale per tile and per key."""

from __future__ import annotations

import numpy as np
import pytest

from long_context_dispatch import Q8, many
from long_context_helpers import Cache, assert_within, attend, attention_q8_call, check, lib

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    check(lib().accel_hip_init())
    yield


@pytest.mark.parametrize("seq,copies", [(40, 320), (1, 12000)])
@pytest.mark.parametrize("block", [4, 32, 64])
@pytest.mark.parametrize("exponent", [-100, 0, 100])
def test_very_small_and_large_values(seq, copies, block, exponent):
    r = np.random.default_rng(51)
    cache = Cache(300, 2, 64, block)
    cache.fill(r, 300)
    cache.scale["v"] *= np.float32(2.0 ** exponent)
    cache.upload()
    q = r.standard_normal((seq, 2, 64)).astype(np.float32)
    want, bound = attend(q, cache.values("k"), cache.values("v"), 300 - seq, 0, 0, None, cache.value_scale(300))
    got = attention_q8_call(many(q, copies, Q8, 300 - seq, 2), cache, 300 - seq)
    assert_within(got[:, ::copies], want, bound, floor=0)


@pytest.mark.parametrize("seq,copies", [(24, 240), (1, 6000)])
@pytest.mark.parametrize("block", [16, 64, 128])
@pytest.mark.parametrize("apart", [90, 120])
def test_a_block_of_large_values_that_counts_for_little(seq, copies, block, apart):
    """Two key tiles' values lie 2^apart above the others' and their scores 2^7 below: a weight of 2^-144, times its
    values next to nothing."""
    r = np.random.default_rng(52)
    cache = Cache(640, 1, 64, block)
    cache.fill(r, 640)
    cache.codes["k"][:, 0, 0] = 64
    cache.codes["k"][128:256, 0, 0] = -64
    cache.scale["k"][:] = 1 / 64
    cache.scale["v"][128 // block:256 // block] *= np.float32(2.0 ** apart)
    cache.upload()
    q = r.standard_normal((seq, 2, 64)).astype(np.float32) / 8
    q[:, :, 0] = 400  # scores of +-50 from this dim: weights e^-100
    want, bound = attend(q, cache.values("k"), cache.values("v"), 640 - seq, 0, 0, None, cache.value_scale(640))
    got = attention_q8_call(many(q, copies, Q8, 640 - seq, 1), cache, 640 - seq)
    assert_within(got[:, ::copies], want, bound)


@pytest.mark.parametrize("seq,copies", [(40, 160), (1, 5300)])
@pytest.mark.parametrize("block", [16, 64])
def test_scales_of_many_magnitudes(seq, copies, block):
    """Blocks whose scales lie apart by up to 2^16 in values, and queries whose rows do by 2^40."""
    r = np.random.default_rng(53)
    cache = Cache(600, 1, 64, block)
    cache.fill(r, 600)
    cache.scale["v"][:] = 2.0 ** r.integers(-16, 1, cache.scale["v"].shape)
    cache.upload()
    q = (r.standard_normal((seq, 3, 64)) * 2.0 ** np.array([-20, 0, 3])[None, :, None]).astype(np.float32)
    q[:, 1, 7] *= 1000
    position = 600 - seq
    want, bound = attend(q, cache.values("k"), cache.values("v"), position, 0, 0, None, cache.value_scale(600))
    got = attention_q8_call(many(q, copies, Q8, position, 1), cache, position)
    assert_within(got[:, ::copies], want, bound)
