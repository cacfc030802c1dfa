"""Grouped integer products whose token tiles go by strips, to the bit."""
import numpy as np
import pytest

import fp8_ref as R
import i8_ref as Q
import i8_strip_cases as S

pytestmark = pytest.mark.gpu
F32, BF16 = 0, 30


@pytest.mark.parametrize("dst_type", [F32, BF16])
@pytest.mark.parametrize("name", S.CASES)
def test_strips_of_several_groups(gpu, name, dst_type):
    """With gathered rows, scattered outputs, and a few rows behind the last group, which are left as they were."""
    counts, rows, k = S.CASES[name]
    rng = np.random.default_rng(len(name) + dst_type)
    used, n_b = sum(counts), 700
    n_rows = used + 5
    m, x = Q.Matrix(rng, len(counts), rows, k, bias=True, distinct=min(3, len(counts))), Q.Tokens(rng, n_b, k)
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    kw = dict(b_rows=rng.integers(0, 2 * n_b, n_rows).astype(np.int32), b_div=2, dst_rows=rng.permutation(n_rows).astype(np.int32))
    got = R.grouped(m, x, n_b, offsets, n_rows, dst_type, n_rows, **kw)
    Q.check(dst_type, got, *Q.grouped_want(m, x, n_b, offsets, n_rows, n_rows, dst_type, **kw))
