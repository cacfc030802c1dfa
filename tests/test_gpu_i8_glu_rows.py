"""The GLU's integer rows in the kernels for many rows, and for the longest ones."""
import pytest

import test_gpu_i8_products as T

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type_id", T.TYPES)
@pytest.mark.parametrize("act", [0, 1])
@pytest.mark.parametrize("rows,width,extra,offset,size", [(513, 2304, 0, 0, 3), (520, 4400, 3, 1, 2), (1100, 1040, 0, 0, 5), (3, 16400, 0, 0, 2), (2, 65536, 1, 1, 2)])
def test_rows_of_every_kernel(gpu, type_id, act, rows, width, extra, offset, size):
    """With the bounds that the other sizes have."""
    T.test_glu_quantize(gpu, type_id, act, rows, width, extra, offset, size)
