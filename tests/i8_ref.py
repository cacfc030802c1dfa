"""Plain forms of the 8-bit integer rows and products. The products are defined to the bit: the sums are exact, and each of the four
roundings behind them is fp32's."""
from __future__ import annotations

import numpy as np

import fp8_ref as R
import vbmoe as vb

I8 = vb.TYPE_I8


def quantize(x):
    """(codes, scales) by the definition, in fp32 steps: 127 x (times 2^-7, and a with it, which changes no bit but keeps large values
    in range), its quotient by a, and that to an integer."""
    x = np.asarray(x).astype(np.float32)
    finite = np.isfinite(x).all(axis=1)
    v = np.where(finite[:, None], x, 0).astype(np.float32)
    a = np.maximum(np.abs(v).max(axis=1), R.LEAST)
    q = (v * np.float32(127 / 128)) / (a * np.float32(2.0 ** -7))[:, None]
    return np.rint(q).astype(np.int8), np.where(finite, a / np.float32(127), np.float32(np.nan)).astype(np.float32)


class Matrix:
    """Device weights of a vbm_weights; the first `distinct` groups repeat."""

    def __init__(self, rng, groups, rows, k, bias=False, distinct=None):
        self.groups, self.rows, self.k, self.distinct = groups, rows, k, distinct or groups
        self.codes = rng.integers(-128, 128, (self.distinct, rows, k)).astype(np.int8)
        self.scale_values = (rng.random((self.distinct, rows)) * 1e-3 + 1e-4).astype(np.float32)
        at = np.arange(groups) % self.distinct
        self.data, self.scales = vb.DeviceBuffer.from_array(self.codes[at]), vb.DeviceBuffer.from_array(self.scale_values[at])
        self.bias_values = rng.standard_normal((groups, rows)).astype(np.float32) if bias else None
        self.bias = vb.DeviceBuffer.from_array(self.bias_values) if bias else None
        self.desc = vb.Weights(I8, self.data.ptr, self.scales.ptr, vb.ptr(self.bias), groups, rows, k)
        self.type_id = I8


class Tokens:
    def __init__(self, rng, n, k):
        self.codes = rng.integers(-127, 128, (n, k)).astype(np.int8)
        self.scale_values = (rng.random(n) * 0.1 + 1e-3).astype(np.float32)
        self.data, self.scales = vb.DeviceBuffer.from_array(self.codes), vb.DeviceBuffer.from_array(self.scale_values)


def outputs(codes, scales, bias, x, x_scales):
    """fp32 outputs [tokens][rows] of one matrix."""
    sums = x.astype(np.float64) @ codes.astype(np.float64).T              # whole numbers below 2^53
    y = sums.astype(np.float32) * (x_scales[:, None] * scales[None, :])
    return y if bias is None else y + bias


def rounded(dst_type, y):
    """fp32 outputs as they come back in dst_type, in float64."""
    with np.errstate(over="ignore"):
        return R.store_as(dst_type, y)[1]


def grouped_want(m, tokens, n_b, offsets, n_rows, n_dst, dst_type, b_rows=None, b_div=1, dst_rows=None):
    y, written = np.zeros((n_dst, m.rows), np.float32), np.zeros(n_dst, bool)
    for g in range(m.groups):
        i = np.arange(max(0, offsets[g]), max(0, min(n_rows, offsets[g + 1])))
        src = i if b_rows is None else np.where(b_rows[i] >= 0, b_rows[i] // b_div, -1)
        d = i if dst_rows is None else dst_rows[i]
        keep = (d >= 0) & (d < n_dst)
        src, d = src[keep], d[keep]
        known = (src >= 0) & (src < n_b)
        s = np.where(known, src, 0)
        e = g % m.distinct
        v = outputs(m.codes[e], m.scale_values[e], m.bias_values[g] if m.bias_values is not None else None, tokens.codes[s], tokens.scale_values[s])
        y[d], written[d] = np.where(known[:, None], v, np.float32(np.nan)), True
    return rounded(dst_type, y), written


def check(dst_type, got, want, written):
    assert R.is_fill(dst_type, got[~written]).all(), "a row that no group lists was written"
    same = (got[written] == want[written]) | (np.isnan(got[written]) & np.isnan(want[written]))
    assert same.all(), (int((~same).sum()), np.argwhere(~same)[:4])
