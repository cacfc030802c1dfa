"""How exactly the FP8 products are summed: terms beside larger ones that cancel, and root mean square errors."""
import numpy as np
import pytest

import fp8_ref as R
import vbmoe as vb

pytestmark = pytest.mark.gpu
F32, F16, BF16, F8 = 0, 1, 30, 256


def dense(codes, ws, x, bs, dst_type):
    """Outputs [tokens][rows] of one FP8 matrix, as float64."""
    d = [vb.DeviceBuffer.from_array(a) for a in (codes, ws, x, bs)]
    tokens, rows = x.shape[0], codes.shape[0]
    dst = vb.DeviceBuffer(tokens * rows * R.SIZE[dst_type])
    vb.call("vbm_mul_mat_fp8", vb.Weights(F8, d[0].ptr, d[1].ptr, None, 1, *codes.shape), d[2].ptr, d[3].ptr, tokens, dst_type, dst.ptr, None)
    vb.call("vbm_stream_synchronize", None)
    return R.load_as(dst_type, dst, (tokens, rows))


@pytest.mark.parametrize("dst_type,tokens,rows", [(F32, 1, 64), (F16, 3, 64), (BF16, 1, 64), (BF16, 10, 72), (F16, 9, 65536 + 16), (BF16, 7, 65536 + 16),
                                                  (F16, 40, 200), (F16, 300, 1100), (F32, 2048, 5200), (F16, 2048, 5200)])
def test_small_terms_beside_large_ones_that_cancel(gpu, dst_type, tokens, rows):
    """448 * 448 - 448 * 448 + 6 * (3.5 * 4) in one group of eight neighbours: 84. The large terms' leading bit is 2^17; sums of fewer than 14
    bits below it would lose the small ones. fp32 sums, each addition off by a step (2^-23) of at most the sum of the magnitudes: 7."""
    k = 128
    w, x = np.zeros((rows, k)), np.zeros((tokens, k))
    w[:, 40:48] = [448, 448, 3.5, 3.5, 3.5, 3.5, 3.5, 3.5]
    x[:, 40:48] = [448, -448, 4, 4, 4, 4, 4, 4]
    nb = -(-rows // 128)
    got = dense(R.e4m3_round(w), np.ones((nb, 1), np.float32), R.e4m3_round(x), np.ones((tokens, 1), np.float32), dst_type)
    y, size = 84.0, 2 * 448.0 ** 2 + 84
    bound = R.sum_bound(F8, F32, k, y, size)
    assert bound < 8
    assert (np.abs(got - y) <= bound + R.HALF_STEP[dst_type] * (y + bound)).all(), (got.min(), got.max())
