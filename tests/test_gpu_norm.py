"""vbm_add_rms_norm_quantize on the GPU against float64."""
import numpy as np
import pytest

import fp8_ref as R
import i8_ref as Q
import vbmoe as vb

pytestmark = pytest.mark.gpu
F32, F16, BF16, F8, I8 = 0, 1, 30, 256, 24
TYPES = [F32, F16, BF16]
# The norm's relative error in fp32: a row's sum of squares is added up by at most 64 additions a lane, 6 across a wave and 15 across
# waves, each off by half a step (2^-24) of a partial sum of positive terms; the root halves it; then the mean, eps, the root, the
# reciprocal and two products: 43 + 6 roundings.
REL = 50 * 2.0 ** -24


def place(raw, stride, offset):
    rows, k = raw.shape
    host = np.zeros(offset + rows * stride, raw.dtype)
    host[offset:].reshape(rows, stride)[:, :k] = raw
    return vb.DeviceBuffer.from_array(host)


def run(type_id, x, residual, weight, eps, y_type, code_type, strides=(None, None), offset=0, in_place=None):
    """(sum, y, codes, scales) of what is asked for, None for the rest; nothing behind them is written."""
    rows, k = x.shape
    xs, rs = (s or k for s in strides)
    es = R.SIZE[type_id]
    dx = place(R.store_as(type_id, x)[0], xs, offset)
    dr = place(R.store_as(type_id, residual)[0], rs, offset) if residual is not None else None
    at = lambda d: d.ptr + offset * es if d is not None else None  # noqa: E731
    d_sum = {None: R.filled((offset + rows * rs) * es + 64) if dr is not None else None, "x": dx, "residual": dr, "no": None}[in_place]
    dw = vb.DeviceBuffer.from_array(weight) if weight is not None else None
    dy = R.filled(rows * k * R.SIZE[y_type] + 64) if y_type is not None else None
    n_scales = rows * (-(-k // 128) if code_type == F8 else 1)
    dc, ds = (R.filled(rows * k + 64), R.filled(4 * n_scales + 64)) if code_type is not None else (None, None)
    vb.call("vbm_add_rms_norm_quantize", type_id, at(dx), xs, at(dr), at(d_sum), rs, vb.ptr(dw), rows, k, eps, y_type or 0, vb.ptr(dy), code_type or 0,
            vb.ptr(dc), vb.ptr(ds), None)
    vb.call("vbm_stream_synchronize", None)
    out = [None] * 4
    if d_sum is not None:
        raw = d_sum.download({F32: np.float32, F16: np.float16, BF16: np.uint16}[type_id], (offset + rows * rs,))[offset:].reshape(rows, rs)
        if in_place is None and rs > k:
            assert (np.ascontiguousarray(raw[:, k:]).view(np.uint8) == R.FILL).all(), "the sum's rows were written past their end"
        out[0] = R.bf16_values(raw[:, :k]) if type_id == BF16 else raw[:, :k].astype(np.float32)
    if dy is not None:
        assert (dy.download(np.uint8, (dy.nbytes,))[-64:] == R.FILL).all()
        out[1] = R.load_as(y_type, dy, (rows, k))
    if dc is not None:
        codes, scales = dc.download(np.uint8, (dc.nbytes,)), ds.download(np.uint8, (ds.nbytes,))
        assert (codes[rows * k:] == R.FILL).all() and (scales[4 * n_scales:] == R.FILL).all()
        out[2], out[3] = codes[:rows * k].reshape(rows, k), scales[:4 * n_scales].view(np.float32).reshape(rows, -1).astype(np.float64)
    return out


def check(type_id, x, residual, weight, eps, y_type, code_type, got):
    x = R.store_as(type_id, x)[1].astype(np.float32)
    if residual is not None:
        x = x + R.store_as(type_id, residual)[1].astype(np.float32)          # rounded to fp32, and then to the type
        x = R.store_as(type_id, x)[1].astype(np.float32)
    total, y, codes, scales = got
    if total is not None:
        assert np.array_equal(total, x)
    v = x.astype(np.float64)
    want = v / np.sqrt((v * v).mean(axis=1, keepdims=True) + float(np.float32(eps)))
    want = want if weight is None else want * weight.astype(np.float64)
    if y is not None:
        err = np.abs(y - want)
        assert (err <= (REL + R.HALF_STEP[y_type] * (1 + REL)) * np.abs(want) + R.LEAST_STEP[y_type]).all(), float((err / np.maximum(np.abs(want), 1e-30)).max())
    if codes is None:
        return
    if code_type == I8:
        a = np.maximum(np.abs(want).max(axis=1, keepdims=True), float(R.LEAST))
        q, step = want * 127 / a, 0.5
        assert (np.abs(scales - a / 127) <= (REL + 2.0 ** -24) * a / 127).all()
        assert (np.abs(codes.view(np.int8) - q) <= 0.5 + 127 * (2 * REL + 2.0 ** -23)).all()
        return
    b = R.blocks_of(want)
    a = np.maximum(np.abs(b).max(axis=2), float(R.LEAST))
    assert (np.abs(scales - a / 448) <= (REL + 2.0 ** -24) * a / 448).all()
    q = b * (448 / a)[:, :, None]
    step = np.exp2(np.floor(np.log2(np.maximum(np.abs(q), 2.0 ** -6)))) / 16
    assert (np.abs(R.blocks_of(R.E4M3[codes]) - q) <= step * (1 + 1e-4) + 448 * (2 * REL + 2.0 ** -23)).all()


SHAPES = [(1, 16), (1, 2880), (5, 128), (9, 512), (6, 528), (3, 2048), (37, 2064), (2, 4096), (5, 4112), (3, 8192), (2, 8208), (2, 16400), (1, 65536), (1500, 208), (600, 2064), (520, 4112)]


@pytest.mark.parametrize("type_id", TYPES)
@pytest.mark.parametrize("code_type", [F8, I8])
@pytest.mark.parametrize("rows,k", SHAPES)
def test_norm(gpu, type_id, code_type, rows, k):
    rng = np.random.default_rng(rows + k)
    x, residual = rng.standard_normal((rows, k)), rng.standard_normal((rows, k)) * 4
    x[:, rng.integers(0, k)] *= 30
    weight = (rng.random(k) + 0.5).astype(np.float32)
    args = (type_id, x, residual, weight, 1e-5, type_id, code_type)
    check(*args, run(*args))


@pytest.mark.parametrize("type_id", TYPES)
@pytest.mark.parametrize("in_place", ["x", "residual", "no"])
@pytest.mark.parametrize("strides,offset", [((None, None), 0), ((2069, 2069), 1), ((2072, 2072), 8)])
def test_sums_in_place_strides_and_alignment(gpu, type_id, in_place, strides, offset):
    rng = np.random.default_rng(offset)
    x, residual = rng.standard_normal((7, 2064)), rng.standard_normal((7, 2064))
    args = (type_id, x, residual, None, 1e-6, F32, F8)
    check(*args, run(*args, strides=strides, offset=offset, in_place=in_place))


@pytest.mark.parametrize("y_type,code_type,with_residual", [(F32, None, True), (BF16, None, False), (None, I8, True), (None, F8, False), (F16, I8, False)])
def test_parts_that_are_not_asked_for(gpu, y_type, code_type, with_residual):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((6, 336))
    args = (BF16, x, rng.standard_normal((6, 336)) if with_residual else None, None, 1e-3, y_type, code_type)
    check(*args, run(*args, strides=(400, 352)))


@pytest.mark.parametrize("code_type", [F8, I8])
def test_small_large_and_zero_rows(gpu, code_type):
    """Rows far below eps, of zeros, and of fp32's large values whose squares still fit."""
    rng = np.random.default_rng(4)
    x = rng.standard_normal((5, 2880)).astype(np.float32)
    x[0] = 0.0
    x[1] *= np.float32(1e-20)
    x[2] *= np.float32(1e15)
    x[3, 1:] = 0.0
    args = (F32, x, None, None, 1e-6, F32, code_type)
    check(*args, run(*args))


@pytest.mark.parametrize("type_id", TYPES)
@pytest.mark.parametrize("code_type", [F8, I8])
@pytest.mark.parametrize("k", [336, 2064])
def test_rows_without_a_norm(gpu, type_id, code_type, k):
    """A NaN, an infinity, a sum that leaves fp16's range, squares that leave fp32's: that row is NaN with codes of zero, its sum stored as
    it is, and no other row is touched by it."""
    rng = np.random.default_rng(6)
    x, residual = rng.standard_normal((8, k)), rng.standard_normal((8, k))
    bad = [1, 3, 5]
    x[1, k - 1] = np.nan
    residual[3, 0] = np.inf
    x[5, 2], residual[5, 2] = {F16: (60000.0, 60000.0), F32: (3e30, 1.0), BF16: (3e30, 1.0)}[type_id]
    with np.errstate(over="ignore", invalid="ignore"):
        total, y, codes, scales = run(type_id, x, residual, None, 1e-6, F32, code_type)
        good = np.setdiff1d(np.arange(8), bad)
        check(type_id, x[good], residual[good], None, 1e-6, F32, code_type, (total[good], y[good], codes[good], scales[good]))
        want = R.store_as(type_id, (R.store_as(type_id, x)[1].astype(np.float32) + R.store_as(type_id, residual)[1].astype(np.float32)))[1]
    assert np.isnan(y[bad]).all() and np.isnan(scales[bad]).all() and (codes[bad] == 0).all()
    same = (total == want) | (np.isnan(total) & np.isnan(want))
    assert same.all()


def test_many_rows(gpu):
    """More rows than workgroups: 1 500 000 of 16 values, each with its own scale."""
    rows, k = 1_500_000, 16
    x = np.tile((np.arange(1000 * k) % 251 - 125).astype(np.float32).reshape(1000, k), (1500, 1))
    _, y, codes, scales = run(F32, x, None, None, 1e-6, F32, I8)
    for part in (y, codes, scales):
        assert np.array_equal(part[:1000], part[-1000:]) and np.array_equal(part[:1000], part[1_048_000:1_049_000])
    check(F32, x[:1000], None, None, 1e-6, F32, I8, (None, y[:1000], codes[:1000], scales[:1000]))
