"""Plain float64 forms of the block-scaled FP8 and the grouped products, and device calls for the tests."""
from __future__ import annotations

import ctypes as C

import numpy as np

import vbmoe as vb

LEAST = np.float32(2.0 ** -116)
F8 = vb.TYPE_F8_E4M3


def e4m3_table():
    codes = np.arange(256)
    s, e, m = codes >> 7, (codes >> 3) & 15, codes & 7
    v = np.where(e > 0, (1 + m / 8.0) * np.exp2(e - 7.0), m / 8.0 * 2.0 ** -6)
    v = np.where(s == 1, -v, v)
    v[(codes & 0x7F) == 0x7F] = np.nan
    return v


E4M3 = e4m3_table()


def e4m3_round(q):
    """Codes of the nearest e4m3 values (|q| <= 448), ties to even."""
    size = np.abs(q.astype(np.float64))
    with np.errstate(divide="ignore"):
        step = np.exp2(np.maximum(np.floor(np.log2(size)), -6.0) - 3)
    v = np.round(size / step) * step                                   # numpy rounds ties to even
    codes = np.searchsorted(E4M3[:127], v)                             # the positive codes' values ascend
    return (codes | np.where(np.signbit(q), 128, 0)).astype(np.uint8)


def blocks_of(x):
    """[rows][k] -> [rows][ceil(k / 128)][128], zeros past the end."""
    rows, k = x.shape
    kb = -(-k // 128)
    v = np.zeros((rows, kb * 128), x.dtype)
    v[:, :k] = x
    return v.reshape(rows, kb, 128)


def quantize(x):
    """(codes, scales) by the definition, in fp32 steps: 448 x, then its quotient by a."""
    x = x.astype(np.float32)
    rows, k = x.shape
    v = blocks_of(x)
    finite = np.isfinite(v).all(axis=2)
    a = np.maximum(np.abs(np.where(finite[:, :, None], v, 0)).max(axis=2), LEAST)
    # (448 x is taken times 2^-9, and a with it, which changes no bit but keeps large values in range)
    q = np.where(finite[:, :, None], (v * np.float32(0.875)) / (a * np.float32(2.0 ** -9))[:, :, None], 0).astype(np.float32)
    codes = np.where(finite[:, :, None], e4m3_round(q), 0).astype(np.uint8)
    scales = np.where(finite, a / np.float32(448.0), np.float32(np.nan)).astype(np.float32)
    return codes.reshape(rows, -1)[:, :k].copy(), scales


def rows_of(codes, scales):
    """float64 values of quantized rows."""
    k = codes.shape[1]
    return E4M3[codes] * scales.astype(np.float64).repeat(128, axis=1)[:, :k]


def fp8_matrix(rng, groups, rows, k):
    """Random e4m3 codes of normal weights and their block scales."""
    nb, kb = -(-rows // 128), -(-k // 128)
    codes = e4m3_round(np.clip(rng.standard_normal((groups, rows, k)) * 120, -448, 448))
    scales = (rng.random((groups, nb, kb)) * 4e-4 + 1e-4).astype(np.float32)
    return codes, scales


def matrix_of(codes, scales):
    groups, rows, k = codes.shape
    s = scales.astype(np.float64).repeat(128, axis=1)[:, :rows].repeat(128, axis=2)[:, :, :k]
    return E4M3[codes] * s


def bf16_bits(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def bf16_values(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32)


def store_as(type_id, x):
    """(array to upload, its float64 values)."""
    if type_id == vb.TYPE_F32:
        a = np.ascontiguousarray(x, np.float32)
        return a, a.astype(np.float64)
    if type_id == vb.TYPE_F16:
        a = np.ascontiguousarray(x, np.float16)
        return a, a.astype(np.float64)
    bits = bf16_bits(x)
    return bits, bf16_values(bits).astype(np.float64)


def load_as(type_id, buf, shape):
    if type_id == vb.TYPE_F32:
        return buf.download(np.float32, shape).astype(np.float64)
    if type_id == vb.TYPE_F16:
        return buf.download(np.float16, shape).astype(np.float64)
    return bf16_values(buf.download(np.uint16, shape)).astype(np.float64)


SIZE = {vb.TYPE_F32: 4, vb.TYPE_F16: 2, vb.TYPE_BF16: 2}
# half a step of the output type, relative to the value (torch.finfo(t).eps / 2)
HALF_STEP = {vb.TYPE_F32: 2.0 ** -24, vb.TYPE_F16: 2.0 ** -11, vb.TYPE_BF16: 2.0 ** -8}
LEAST_STEP = {vb.TYPE_F32: 0.0, vb.TYPE_F16: 2.0 ** -25, vb.TYPE_BF16: 0.0}   # half a subnormal step of fp16


class Matrix:
    """Device weights of a vbm_weights, and the float64 values of their first `distinct` groups, which repeat."""

    def __init__(self, type_id, rng, groups, rows, k, bias=False, distinct=None):
        self.type_id, self.groups, self.rows, self.k, self.distinct = type_id, groups, rows, k, distinct or groups
        repeated = lambda a: vb.DeviceBuffer.from_array(a[np.arange(groups) % self.distinct])  # noqa: E731
        if type_id == F8:
            codes, scales = fp8_matrix(rng, self.distinct, rows, k)
            self.values = matrix_of(codes, scales)
            self.data, self.scales = repeated(codes), repeated(scales)
        else:
            raw, self.values = store_as(type_id, rng.standard_normal((self.distinct, rows, k)) / np.sqrt(k))
            self.data, self.scales = repeated(raw), None
        self.bias_values = rng.standard_normal((groups, rows)).astype(np.float32) * np.float32(0.1) if bias else None
        self.bias = vb.DeviceBuffer.from_array(self.bias_values) if bias else None
        self.desc = vb.Weights(type_id, self.data.ptr, vb.ptr(self.scales), vb.ptr(self.bias), groups, rows, k)


class Tokens:
    """Device token rows in the weights' type, and their float64 values."""

    def __init__(self, type_id, rng, n, k):
        x = rng.standard_normal((n, k)).astype(np.float32)
        if type_id == F8:
            codes, scales = quantize(x)
            self.values = rows_of(codes, scales)
            self.data, self.scales = vb.DeviceBuffer.from_array(codes), vb.DeviceBuffer.from_array(scales)
        else:
            raw, self.values = store_as(type_id, x)
            self.data, self.scales = vb.DeviceBuffer.from_array(raw), None


def sum_bound(type_id, dst_type, k, y, size):
    """How far an output may be from its float64 value y, `size` being the sum of its terms' magnitudes. The
    products are exact in fp32; k of them, the blocks' sums and the bias are added in fp32, each addition off by at most a step
    (2^-23, where the matrix core cuts off instead of rounding) of a partial sum that is no larger than `size`; an
    FP8 block's sum also takes the rounded product of its two scales and one more rounding. For 16-bit outputs of FP8
    weights the matrix core adds eight products at a time, cut off 13 bits below the leading bit of the largest: seven of them lose at
    most 2^-13 of it each, and it is no larger than the eight's magnitudes' sum. Then one rounding to dst_type."""
    adds = k + 2 * -(-k // 128) + 16
    err = adds * 2.0 ** -23 * size
    if type_id == F8 and dst_type != vb.TYPE_F32:
        err = err + 7 * 2.0 ** -13 * size
    return err + HALF_STEP[dst_type] * (np.abs(y) + err) + LEAST_STEP[dst_type]


FILL = 0x5A


def filled(nbytes):
    """A device buffer of FILL bytes: what a call leaves alone keeps them."""
    return vb.DeviceBuffer.from_array(np.full(nbytes, FILL, np.uint8))


def is_fill(type_id, values):
    if type_id == vb.TYPE_F32:
        return values == float(np.full(4, FILL, np.uint8).view(np.float32)[0])
    if type_id == vb.TYPE_F16:
        return values == float(np.full(2, FILL, np.uint8).view(np.float16)[0])
    return values == float(bf16_values(np.full(2, FILL, np.uint8).view(np.uint16))[0])


def grouped(m, tokens, n_b, offsets, n_rows, dst_type, n_dst, b_rows=None, b_div=1, dst_rows=None, stream=None):
    dev = lambda a: vb.DeviceBuffer.from_array(np.asarray(a, np.int32)) if a is not None else None  # noqa: E731
    d_off, d_b, d_dst = dev(offsets), dev(b_rows), dev(dst_rows)
    dst = filled(n_dst * m.rows * SIZE[dst_type])
    vb.call("vbm_grouped_mul_mat", m.desc, tokens.data.ptr, vb.ptr(tokens.scales), n_b, vb.ptr(d_b), b_div, d_off.ptr, n_rows,
            vb.ptr(d_dst), n_dst, dst_type, dst.ptr, stream)
    vb.call("vbm_stream_synchronize", stream)
    return load_as(dst_type, dst, (n_dst, m.rows))


def grouped_want(m, tokens, n_b, offsets, n_rows, n_dst, b_rows=None, b_div=1, dst_rows=None):
    """(values, sums of magnitudes, written) of dst; NaN where the b row is out of range."""
    y, size, written = np.zeros((n_dst, m.rows)), np.zeros((n_dst, m.rows)), np.zeros(n_dst, bool)
    for g in range(m.groups):
        i = np.arange(max(0, offsets[g]), max(0, min(n_rows, offsets[g + 1])))
        src = i if b_rows is None else np.where(b_rows[i] >= 0, b_rows[i] // b_div, -1)
        d = i if dst_rows is None else dst_rows[i]
        keep = (d >= 0) & (d < n_dst)
        src, d = src[keep], d[keep]
        known = (src >= 0) & (src < n_b)
        x = tokens.values[np.where(known, src, 0)]
        w = m.values[g % m.distinct]
        v, s = x @ w.T, np.abs(x) @ np.abs(w).T
        if m.bias_values is not None:
            v, s = v + m.bias_values[g], s + np.abs(m.bias_values[g])
        y[d], size[d], written[d] = np.where(known[:, None], v, np.nan), s, True
    return y, size, written


def check(m, dst_type, got, y, size, written, name=""):
    assert is_fill(dst_type, got[~written]).all(), "a row that no group lists was written"
    nan = np.isnan(y)
    assert np.isnan(got[nan]).all() and not np.isnan(got[written & ~nan.any(axis=1)]).any()
    ok = written & ~nan.any(axis=1)
    err, bound = np.abs(got[ok] - y[ok]), sum_bound(m.type_id, dst_type, m.k, y[ok], size[ok])
    if err.size:
        print(f"[{name}] worst error / bound {np.max(err / np.maximum(bound, 1e-300)):.3f}", flush=True)
    assert (err <= bound).all(), (float(np.max(err / bound)), np.argwhere(err > bound)[:4])
