"""Offsets that are not in order: the products stay inside their buffers, and the first tiles are done."""
import numpy as np
import pytest

import fp8_ref as R
import vbmoe as vb

pytestmark = pytest.mark.gpu
F32, F8 = 0, 256


@pytest.mark.parametrize("n_rows,groups", [(2000, 8), (60, 64), (4000, 300), ((1 << 29) - 1, 1024)])
def test_groups_that_overlap(gpu, n_rows, groups):
    """Every other group spans all rows, far more tiles than rows in order can have (2^31 in the last case, where the tokens and the outputs
    are those of the first 40 rows). All groups have the same weights, so that the rows' results are the same whoever writes them."""
    rng = np.random.default_rng(groups)
    rows, k, n = 16, 16, 40
    m, x = R.Matrix(F8, rng, groups, rows, k, distinct=1), R.Tokens(F8, rng, n, k)
    offsets = np.where(np.arange(groups + 1) % 2, n_rows, 0).astype(np.int32)
    d_off, dst = vb.DeviceBuffer.from_array(offsets), R.filled((n + 4) * rows * 4)
    vb.call("vbm_grouped_mul_mat", m.desc, x.data.ptr, x.scales.ptr, n, None, 1, d_off.ptr, n_rows, None, n, F32, dst.ptr, None)
    vb.call("vbm_stream_synchronize", None)
    got = R.load_as(F32, dst, (n + 4, rows))
    assert R.is_fill(F32, got[n:]).all()
    y = x.values @ m.values[0].T
    bound = R.sum_bound(F8, F32, k, y, np.abs(x.values) @ np.abs(m.values[0]).T)
    assert (np.abs(got[:n] - y) <= bound).all()
