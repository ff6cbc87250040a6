"""Plain 64-bit forms of the long-context operators, and the bounds their tests use."""

from __future__ import annotations

import ctypes as C

import numpy as np

from accelep_amd import capi
from accelep_amd.capi import Buffer, CacheQ8, check, lib
from accelep_amd.device import DeviceArray
from hip_helpers import dev

NONE = Buffer(None, 0, 0)
U = 2.0 ** -24


def nearest(x):
    return np.rint(x)  # ties to even


class Cache:
    """An 8-bit cache on the device beside its plain form: codes and scales as appended so far."""

    def __init__(self, capacity, kv_heads, dim, block):
        self.shape = (capacity, kv_heads, dim)
        self.block = block
        blocks = -(-capacity // block)
        self.codes = {n: np.zeros(self.shape, np.int8) for n in "kv"}
        self.scale = {n: np.zeros((blocks, kv_heads), np.float32) for n in "kv"}
        self.d_codes = {n: dev(self.codes[n]) for n in "kv"}
        self.d_scale = {n: dev(self.scale[n]) for n in "kv"}
        self.handle = CacheQ8(self.d_codes["k"].buffer, self.d_codes["v"].buffer, self.d_scale["k"].buffer,
                              self.d_scale["v"].buffer, capacity, kv_heads, dim, block)

    def fill(self, rng, rows, spread=0.5):
        """Rows already there: any codes, scales of a few magnitudes."""
        for n in "kv":
            self.codes[n][:rows] = rng.integers(-127, 128, (rows, *self.shape[1:]), dtype=np.int8)
            self.scale[n][:] = np.exp(spread * rng.standard_normal(self.scale[n].shape)) / 64
            self.upload()

    def upload(self):
        for n in "kv":
            self.d_codes[n].upload(self.codes[n])
            self.d_scale[n].upload(self.scale[n])

    def append(self, k, v, position):
        """The plain form, block by block, in 64 bits (a scale is held in 32)."""
        for n, x in (("k", k), ("v", v)):
            x = np.asarray(x, np.float64)
            seq, B = len(x), self.block
            for b in range(position // B, (position + seq - 1) // B + 1 if seq else 0):
                begin = b * B
                lo, hi = max(position, begin), min(position + seq, begin + B)
                new = x[lo - position:hi - position]
                need = (np.abs(new).max(axis=(0, 2)) / 127).astype(np.float32)
                need[~np.isfinite(new).all(axis=(0, 2))] = np.nan
                old = self.scale[n][b].copy() if lo > begin else np.zeros_like(need)
                now = np.maximum(need, old)  # a NaN on either side stays one
                kept = self.codes[n][begin:lo]
                with np.errstate(invalid="ignore", divide="ignore"):
                    again = nearest(kept * old.astype(np.float64)[None, :, None] / now.astype(np.float64)[None, :, None])
                    # (a scale below 2^-126 has few bits: its codes may pass 127 and stay there)
                    code = np.clip(nearest(new / now.astype(np.float64)[None, :, None]), -127, 127)
                grows = now > old
                self.codes[n][begin:lo] = np.where(grows[None, :, None], again, kept)
                self.codes[n][lo:hi] = np.nan_to_num(np.where((now > 0)[None, :, None], code, 0))
                self.scale[n][b] = now

    def values(self, n):
        """fp32 values, code * scale rounded once."""
        with np.errstate(invalid="ignore"):
            by_row = np.repeat(self.scale[n], self.block, axis=0)[:self.shape[0], :, None]
            return (self.codes[n].astype(np.float32) * by_row).astype(np.float32)

    def value_scale(self, rows):
        return np.repeat(self.scale["v"], self.block, axis=0)[:rows]

    def on_device(self):
        return ({n: self.d_codes[n].numpy() for n in "kv"}, {n: self.d_scale[n].numpy() for n in "kv"})


def append_call(cache, k, v, position, row_stride=0):
    kd, vd = dev(np.asarray(k, np.float32)), dev(np.asarray(v, np.float32))
    check(lib().accel_hip_append_cache_q8(kd.buffer, vd.buffer, C.byref(cache.handle), len(k), position, row_stride))
    return kd, vd


def sees(position, seq, rows, window, sinks):
    """[seq, rows] truth values: which keys each row sees."""
    p = position + np.arange(seq)[:, None]
    t = np.arange(rows)[None, :]
    seen = t <= p
    if window:
        seen &= (t > p - window) | (t < sinks)
    return seen


def attend(q, k, v, position, window, sinks, rows=None, value_scale=None):
    """(out, bound) in 64 bits: softmax attention of the rows `rows` (all), and how far fp32 sums may be off.

    A score is a dot of D products, each off by U with either sign, and so is its sum: 8 sqrt(D) U sum|q k|
    (the probabilistic bound, at 8 standard deviations), plus the 22-bit query (4 U of the same sum) and the
    exponent's rounding (4 U (1 + |s|)). A weight is off by that, twice (numerator and sum), and the weighted
    sums over n keys by 8 sqrt(n) U each, and 4 U for the 22-bit weight; the quotient adds 2 U.

    value_scale [rows, kv_heads], for the 8-bit cache: the 22 bits of a weight are relative to the largest. A weight
    enters as w = p * scale * 2^e with the largest w of the row in [2^3, 2^15), in two f16 parts cut towards zero:
    off by 2^-22 w where the second part is a normal number, and by less than the spacing of f16's subnormal ones,
    2^-24, where it is not, which is 2^-27 of the largest w. So a key adds at most 2^-27 max(p * scale) |code|."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    seq, heads, dim = q.shape
    group = heads // k.shape[1]
    rows = np.arange(seq) if rows is None else np.asarray(rows)
    out, bound = np.empty((len(rows), heads, dim)), np.empty((len(rows), heads, dim))
    seen = sees(position, seq, position + seq, window, sinks)
    for i, s in enumerate(rows):
        at = np.flatnonzero(seen[s])
        for h in range(heads):
            kk, vv = k[at, h // group], v[at, h // group]
            x = kk @ q[s, h] / np.sqrt(dim)
            spread = np.abs(kk) @ np.abs(q[s, h]) / np.sqrt(dim)
            e = np.exp(x - x.max())
            p = e / e.sum()
            d = (8 * np.sqrt(dim) + 4) * U * spread + 4 * U * (1 + np.abs(x) + np.abs(x.max()))
            out[i, h] = p @ vv
            share = p * (d + 16 * np.sqrt(len(at)) * U + 6 * U)
            bound[i, h] = share @ np.abs(vv) + share.sum() * np.abs(out[i, h])
            if value_scale is not None:
                scale = np.asarray(value_scale, np.float64)[at, h // group]
                bound[i, h] += 2.0 ** -27 * (p * scale).max() * (np.abs(vv) / scale[:, None]).sum(axis=0)
    return out, bound


def assert_within(got, want, bound, floor=1e-30):
    err = np.abs(np.asarray(got, np.float64) - want)
    bad = ~(err <= bound + floor)
    if bad.any():
        at = tuple(np.argwhere(bad)[0])
        near = np.sort(np.where(np.isfinite(err), err, 0).ravel())[-8:]
        raise AssertionError(f"{bad.sum()} of {bad.size} beyond the bound; first at {at}: {got[at]!r}, {want[at]!r} wanted, "
                             f"bound {np.broadcast_to(bound, err.shape)[at]:.3g}; largest errors {near}")


def attention_q8_call(q, cache, position, window=0, sinks=0, row_stride=0, shape=None):
    """shape: (seq, heads, dim) of a q whose rows are row_stride apart."""
    shape = q.shape if shape is None else shape
    out = dev(np.full(shape, 3.0, np.float32))
    qd = dev(np.asarray(q, np.float32))
    check(lib().accel_hip_attention_q8(qd.buffer, C.byref(cache.handle), out.buffer, shape[0], position, shape[1],
                                       row_stride, window, sinks))
    return out.numpy()


def attention_window_call(q, k, v, position, window=0, sinks=0, row_stride=0, shape=None):
    shape = q.shape if shape is None else shape
    out = dev(np.full(shape, 3.0, np.float32))
    qd, kd, vd = (dev(np.asarray(x, np.float32)) for x in (q, k, v))
    check(lib().accel_hip_attention_window(qd.buffer, kd.buffer, vd.buffer, out.buffer, shape[0], position, shape[1],
                                           k.shape[1], shape[2], row_stride, window, sinks))
    return out.numpy()


def frequencies(kind, rotary, theta=1e5, factor=8.0, original=4096.0, fast=32.0, slow=1.0):
    i = np.arange(rotary // 2, dtype=np.float64)
    f = theta ** (-2 * i / rotary)
    if kind == capi.ROPE_SCALE_LINEAR:
        return f / factor
    if kind == capi.ROPE_SCALE_NTK:
        return (theta * factor ** (rotary / (rotary - 2))) ** (-2 * i / rotary)
    if kind == capi.ROPE_SCALE_YARN:
        # pairs by the turns they make over the original context, theta^(-2i/r) L / 2 pi
        pair = lambda n: rotary * np.log(original / (2 * np.pi * n)) / (2 * np.log(theta))  # noqa: E731
        low, high = max(np.floor(pair(fast)), 0), min(np.ceil(pair(slow)), rotary - 1)
        divided = np.clip((i - low) / max(high - low, 1e-3), 0, 1)
        return f * (1 - divided) + f / factor * divided
    if kind == capi.ROPE_SCALE_WAVELENGTH:
        left = np.clip((original * f / (2 * np.pi) - slow) / (fast - slow), 0, 1)
        return f * left + f / factor * (1 - left)
    return f


def rotated(x, f, positions, layout, magnitude):
    """(values, bound) of [seq, heads, dim] rows in 64 bits. cos and sin come from a library's sincospi (4 ulp,
    4 U of 1 at most) with three more roundings of U and the magnitude's; a product and the sum add one each."""
    x = np.asarray(x, np.float64)
    r = 2 * len(f)
    first, second = (np.arange(r // 2), np.arange(r // 2) + r // 2) if layout == capi.ROPE_HALF else (
        2 * np.arange(r // 2), 2 * np.arange(r // 2) + 1)
    a = np.asarray(positions, np.float64)[:, None, None] * f
    out, bound = x.copy(), np.zeros_like(x)
    x0, x1 = x[..., first], x[..., second]
    out[..., first] = magnitude * (x0 * np.cos(a) - x1 * np.sin(a))
    out[..., second] = magnitude * (x1 * np.cos(a) + x0 * np.sin(a))
    bound[..., first] = bound[..., second] = 10 * U * magnitude * (np.abs(x0) + np.abs(x1))
    return out, bound


__all__ = ["Cache", "DeviceArray", "NONE", "U", "append_call", "assert_within", "attend", "attention_q8_call",
           "attention_window_call", "capi", "check", "dev", "frequencies", "lib", "rotated", "sees"]
