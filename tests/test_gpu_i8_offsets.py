"""Integer products whose offsets are not in order, and weights past 2^32 bytes, there and in the layer for a few tokens."""
import ctypes as C

import numpy as np
import pytest

import fp8_ref as R
import i8_ref as Q
import vbmoe as vb

pytestmark = pytest.mark.gpu
F32, I8 = 0, 24


@pytest.mark.parametrize("n_rows,groups", [(2000, 8), (60, 64), (4000, 300), (60000, 3), ((1 << 29) - 1, 1024)])
def test_groups_that_overlap(gpu, n_rows, groups):
    """Every other group spans all rows, far more tiles than rows in order can have. All groups have the same weights, so that the rows'
    results are the same whoever writes them."""
    rng = np.random.default_rng(groups)
    rows, k, n = 16, 16, 40
    m, x = Q.Matrix(rng, groups, rows, k, distinct=1), Q.Tokens(rng, n, k)
    offsets = np.where(np.arange(groups + 1) % 2, n_rows, 0).astype(np.int32)
    d_off, dst = vb.DeviceBuffer.from_array(offsets), R.filled((n + 4) * rows * 4)
    vb.call("vbm_grouped_mul_mat", m.desc, x.data.ptr, x.scales.ptr, n, None, 1, d_off.ptr, n_rows, None, n, F32, dst.ptr, None)
    vb.call("vbm_stream_synchronize", None)
    got = R.load_as(F32, dst, (n + 4, rows))
    assert R.is_fill(F32, got[n:]).all()
    assert np.array_equal(got[:n], Q.outputs(m.codes[0], m.scale_values[0], None, x.codes, x.scale_values))


def ones(n):
    buf = vb.DeviceBuffer(n)
    vb.call("vbm_memset", buf.ptr, 1, n, None)
    return buf


@pytest.mark.parametrize("tokens", [1, 30, 300])
def test_weights_past_four_gigabytes(gpu, tokens):
    """All weights are 1 but for one row of the last group, behind 5 GB."""
    rng = np.random.default_rng(tokens)
    groups, rows, k = 41, 1000, 131056
    w = ones(groups * rows * k)
    special = rng.integers(-128, 128, k).astype(np.int8)
    vb.call("vbm_memcpy_h2d", w.ptr + (groups * rows - 3) * k, special.ctypes.data, k, None)
    x, scales = Q.Tokens(rng, tokens, k), rng.random((groups, rows)).astype(np.float32)
    ds = vb.DeviceBuffer.from_array(scales)
    offsets = np.zeros(groups + 1, np.int32)
    offsets[-1] = tokens
    d_off, dst = vb.DeviceBuffer.from_array(offsets), vb.DeviceBuffer(tokens * rows * 4)
    vb.call("vbm_grouped_mul_mat", vb.Weights(I8, w.ptr, ds.ptr, None, groups, rows, k), x.data.ptr, x.scales.ptr, tokens, None, 1, d_off.ptr, tokens,
            None, tokens, F32, dst.ptr, None)
    vb.call("vbm_stream_synchronize", None)
    sums = np.repeat(x.codes.astype(np.int64).sum(axis=1)[:, None], rows, axis=1)
    sums[:, -3] = x.codes.astype(np.int64) @ special.astype(np.int64)
    want = sums.astype(np.float32) * (x.scale_values[:, None] * scales[-1][None, :])
    assert np.array_equal(dst.download(np.float32, (tokens, rows)), want)


def test_layer_weights_past_four_gigabytes(gpu):
    """All weights are 1 but for a gate and an up row and a down row of the last expert: gate_up is 4.8 GB, down 2.4. The scales keep gate and up near 1.
    The sums of 65536 and 4096 products are off by at most as many steps (2^-23) of their magnitudes; the GLU passes on twice as much here."""
    rng = np.random.default_rng(3)
    E, H, I, T = 9, 65536, 4096, 2
    gu, dn = ones(E * 2 * I * H), ones(E * H * I)
    gate, up, down = (rng.integers(-128, 128, n).astype(np.int8) for n in (H, H, I))
    vb.call("vbm_memcpy_h2d", gu.ptr + ((E - 1) * 2 * I + I - 1) * H, gate.ctypes.data, H, None)
    vb.call("vbm_memcpy_h2d", gu.ptr + (E * 2 * I - 1) * H, up.ctypes.data, H, None)
    vb.call("vbm_memcpy_h2d", dn.ptr + (E * H - 1) * I, down.ctypes.data, I, None)
    s1, s2 = np.full((E, 2 * I), 2.0 ** -10, np.float32), np.full((E, H), 2.0 ** -6, np.float32)
    x = rng.standard_normal((T, H)).astype(np.float32)
    ids, weights = np.full((T, 1), E - 1, np.int32), np.ones((T, 1), np.float32)
    d = [vb.DeviceBuffer.from_array(a) for a in (s1, s2, x, ids, weights)]
    desc = vb.MoeFewDesc(vb.Weights(I8, gu.ptr, d[0].ptr, None, E, 2 * I, H), vb.Weights(I8, dn.ptr, d[1].ptr, None, E, H, I), 1, 0, 1.0, 1.0)
    size = C.c_size_t()
    vb.call("vbm_moe_few_workspace", desc, T, size)
    ws, out = vb.DeviceBuffer(size.value), vb.DeviceBuffer(T * H * 4)
    vb.call("vbm_moe_few_forward", desc, F32, d[2].ptr, None, d[3].ptr, d[4].ptr, T, F32, out.ptr, ws.ptr, size.value, None)
    vb.call("vbm_stream_synchronize", None)
    got = out.download(np.float32, (T, H)).astype(np.float64)
    for t in range(T):
        v = x[t].astype(np.float64)
        g, u = np.full(I, v.sum()), np.full(I, v.sum())
        g[-1], u[-1] = gate @ v, up @ v
        size_g = np.full(I, np.abs(v).sum())
        size_g[-1] = max(np.abs(gate.astype(np.float64)) @ np.abs(v), np.abs(up.astype(np.float64)) @ np.abs(v))
        g, u, err = g * 2.0 ** -10, u * 2.0 ** -10, 6 * H * 2.0 ** -23 * size_g * 2.0 ** -10
        h = g / (1 + np.exp(-g)) * u
        dh = 1.1 * (np.abs(u) + 1) * err + np.abs(g) * err + (np.abs(g) + 8) * 2.0 ** -24 * np.abs(h)
        for row, w in ((0, np.ones(I)), (H - 2, np.ones(I)), (H - 1, down.astype(np.float64))):
            bound = 2.0 ** -6 * (np.abs(w) @ dh + 6 * I * 2.0 ** -23 * (np.abs(w) @ np.abs(h)))
            assert abs(got[t, row] - 2.0 ** -6 * (w @ h)) <= bound, (t, row, got[t, row], 2.0 ** -6 * (w @ h), bound)
            # (random signs: far closer than all errors at once)
            assert abs(got[t, row] - 2.0 ** -6 * (w @ h)) <= 2e-4 * 2.0 ** -6 * (np.abs(w) @ np.abs(h))
        assert (got[t, :-1] == got[t, 0]).all()
