"""Where the residual norm may leave its sum, before any device is touched: x's buffer takes it only row for row."""
import pytest

import test_i8_products as T

A = 4096                                        # an aligned address that nothing here dereferences
ROWS = dict(T.NORM, x=A, sum=A, x_stride=256, residual_stride=128, k=128)


@pytest.mark.parametrize("change", [{}, dict(residual=2 * A), dict(x_stride=128, residual_stride=256, residual=2 * A), dict(n_rows=2)])
def test_sum_in_rows_that_other_rows_still_read(vb, change):
    """With other strides a row's sum lands in rows of x that another workgroup has yet to read."""
    T.refused(vb, b"x's buffer", "vbm_add_rms_norm_quantize", *{**ROWS, **change}.values())


@pytest.mark.parametrize("change", [dict(residual_stride=256), dict(n_rows=1), dict(sum=2 * A), dict(n_rows=0)])
def test_sums_that_are_in_nobodys_way(vb, change):
    """These pass the buffers' checks: what is refused is the codes' type, which is looked at behind them."""
    T.refused(vb, b"F8_E4M3 or I8", "vbm_add_rms_norm_quantize", *{**ROWS, "residual": 2 * A, "code_type": T.F16, **change}.values())
