"""vbm_glu_quantize_fp8 at gates whose exponentials leave the fp32 range."""
import numpy as np
import pytest

import fp8_ref as R
import vbmoe as vb

pytestmark = pytest.mark.gpu
F32, BF16 = 0, 30
# The largest fp32 value whose exponential rounds to one too: that has to stay below 2^128 (1 - 2^-25), whose logarithm is
# 128 ln 2 - 2^-25 = 88.72283908. fp32 values there are 2^-17 apart: 88.72283173 is below it, the next one, NEAR, above.
LAST, NEAR = 88.7228318, np.float32(88.7228394)


def glu_fp32_range(act, g, u, alpha, limit):
    """The definition in float64, with an infinite exponential where fp32's is."""
    if act == 1:
        g, u = np.minimum(g, limit), np.clip(u, -limit, limit) + 1
    x = -(alpha if act == 1 else 1.0) * g
    e = np.where(x > LAST, np.inf, np.exp(np.minimum(x, 100.0)))
    return g / (1 + e) * u


def run(act, type_id, x, alpha, limit):
    rows, width = x.shape[0], x.shape[1] // 2
    raw, v = R.store_as(type_id, x)
    kb, es = -(-width // 128), R.SIZE[type_id]
    dx, dc, ds = vb.DeviceBuffer.from_array(raw), vb.DeviceBuffer(rows * width), vb.DeviceBuffer(4 * rows * kb)
    vb.call("vbm_glu_quantize_fp8", act, type_id, dx.ptr, dx.ptr + width * es, rows, width, 2 * width, 2 * width, alpha, limit, dc.ptr, ds.ptr, None)
    vb.call("vbm_stream_synchronize", None)
    return v[:, :width], v[:, width:], dc.download(np.uint8, (rows, width)), ds.download(np.float32, (rows, kb)).astype(np.float64)


def check(h, codes, scales):
    """Scales within the fp32 arithmetic's error (the argument's rounding, 104 * 2^-24, and eight more), codes within half a step of e4m3 more."""
    a = np.maximum(np.abs(R.blocks_of(h)).max(axis=2), float(R.LEAST))
    rel = (104 + 8) * 2.0 ** -24
    assert np.isfinite(scales).all()
    assert (np.abs(scales - a / 448) <= rel * a / 448).all(), np.argwhere(np.abs(scales - a / 448) > rel * a / 448)[:4]
    q = R.blocks_of(h) * (448 / a)[:, :, None]
    half = np.exp2(np.floor(np.log2(np.maximum(np.abs(q), 2.0 ** -6)))) / 16
    assert (np.abs(R.blocks_of(R.E4M3[codes]) - q) <= half * (1 + 1e-4) + 2 * rel * 448).all()


GATES = [200.0, 1e10, 1e30, 8.5e37, 1e38, 2.3e38, 2.4e38, 3e38, 3.38e38]


@pytest.mark.parametrize("type_id", [F32, BF16])
@pytest.mark.parametrize("act,limit", [(0, 7.0), (1, 7.0), (1, 1e38)])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_large_finite_gates(gpu, type_id, act, limit, sign):
    """One gate a row, and in the last rows all of them: a large negative one comes out as 0, a large positive one as itself, each times up, and
    neither takes the block's scale away."""
    rng = np.random.default_rng(9)
    width = 144
    x = rng.standard_normal((len(GATES) + 2, 2 * width)).astype(np.float32)
    x[:, width:] = np.clip(x[:, width:], -0.4, 0.4)
    for i, g in enumerate(GATES):
        x[i, 5], x[i, 130] = sign * g, sign * g
    x[-2, :width] = sign * np.resize(GATES, width)
    x[-1, :width] = sign * 3e38
    with np.errstate(over="ignore"):
        g, u, codes, scales = run(act, type_id, x, 1.702, limit)
        check(glu_fp32_range(act, g, u, float(np.float32(1.702)), float(np.float32(limit))), codes, scales)


@pytest.mark.parametrize("act,alpha", [(0, 0.0), (1, 1.0), (1, 1.702), (1, -1.0)])
def test_gates_about_the_end_of_the_exponential(gpu, act, alpha):
    """Arguments from 86 to 90 in fp32 steps about the last one, with ups that bring the products to ordinary size."""
    width = 1024
    x = np.zeros((4, 2 * width), np.float32)
    arg = np.concatenate([np.linspace(86, 90, width - 64), NEAR + np.arange(-32, 32) * np.float32(2.0 ** -17)]).astype(np.float32)
    g = -arg if act == 0 else (-arg / np.float32(alpha)).astype(np.float32)
    if act == 1 and alpha == 1.702:                                       # (their fp32 product is the argument, which may lie on either side)
        g = g[np.abs(arg - NEAR) > 1e-4]
        g = np.resize(g, width)
    x[:, :width] = g
    x[:, width:] = np.array([1e36, -1e36, 3e35, 1e33], np.float32)[:, None]
    gv, u, codes, scales = run(act, F32, x, alpha, 1e36)
    check(glu_fp32_range(act, gv, u, float(np.float32(alpha)), float(np.float32(1e36))), codes, scales)


@pytest.mark.parametrize("act", [0, 1])
def test_infinite_and_nan_gates_have_no_scale(gpu, act):
    width = 128
    x = np.ones((4, 2 * width), np.float32)
    x[0, 3], x[1, 3], x[2, 3] = -np.inf, np.nan, np.inf
    _, _, codes, scales = run(act, F32, x, 1.702, np.inf)
    assert np.array_equal(np.isnan(scales[:, 0]), [True, True, True, False]) and (codes[:3] == 0).all() and (codes[3] == 0x7E).all()
