"""vbm_add_rms_norm_quantize on the GPU: more rows than workgroups where waves share a row, and buffers that are aligned to their type only, one at a time."""
import numpy as np
import pytest

import fp8_ref as R
import vbmoe as vb
from test_gpu_norm import check, run

pytestmark = pytest.mark.gpu
F32, F16, BF16, F8, I8 = 0, 1, 30, 256, 24


def test_more_rows_than_workgroups_where_waves_share_a_row(gpu):
    """1 051 000 rows of 528 values, a thousand of them over and over: a workgroup's second row finds its LDS as the first one left it."""
    times, k = 1051, 528
    rng = np.random.default_rng(8)
    x = (rng.standard_normal((1000, k)) * np.exp2(rng.integers(-6, 6, (1000, 1)))).astype(np.float32)
    _, _, codes, scales = run(F16, np.tile(x, (times, 1)), None, None, 1e-6, None, I8)
    codes, scales = codes.reshape(times, 1000, k), scales.reshape(times, 1000, 1)
    assert (codes == codes[0]).all() and (scales == scales[0]).all()
    check(F16, x, None, None, 1e-6, None, I8, (None, None, codes[0], scales[0]))


@pytest.mark.parametrize("type_id", [F32, F16, BF16])
@pytest.mark.parametrize("code_type", [F8, I8])
@pytest.mark.parametrize("rows,k", [(5, 176), (3, 2064), (520, 2064), (2, 16400)])
def test_buffers_that_are_aligned_to_their_type_only(gpu, type_id, code_type, rows, k):
    """Each in turn an element past an aligned address: the same bits as from aligned ones."""
    rng = np.random.default_rng(k + rows)
    raw = {n: R.store_as(type_id, rng.standard_normal((rows, k)))[0] for n in ("x", "residual")}
    raw["weight"] = (rng.random(k) + 0.5).astype(np.float32)
    es = R.SIZE[type_id]
    size = {"sum": rows * k * es, "y": rows * k * es, "codes": rows * k, "scales": 4 * rows * (-(-k // 128) if code_type == F8 else 1)}

    def call(moved):
        at = {n: (4 if n in ("weight", "scales") else es) if n == moved else 0 for n in (*raw, *size)}
        dev = {n: vb.DeviceBuffer.from_array(np.concatenate([np.full(at[n], R.FILL, np.uint8), np.ascontiguousarray(a).reshape(-1).view(np.uint8)])) for n, a in raw.items()}
        dev.update({n: R.filled(at[n] + b + 64) for n, b in size.items()})
        p = {n: d.ptr + at[n] for n, d in dev.items()}
        vb.call("vbm_add_rms_norm_quantize", type_id, p["x"], k, p["residual"], p["sum"], k, p["weight"], rows, k, 1e-5, type_id, p["y"], code_type,
                p["codes"], p["scales"], None)
        vb.call("vbm_stream_synchronize", None)
        out = {n: dev[n].download(np.uint8, (dev[n].nbytes,)) for n in size}
        assert all((out[n][:at[n]] == R.FILL).all() and (out[n][at[n] + size[n]:] == R.FILL).all() for n in size), moved
        return {n: out[n][at[n]:at[n] + size[n]] for n in size}

    want = call(None)
    for moved in ("x", "residual", "sum", "weight", "y", "scales"):
        got = call(moved)
        assert all(np.array_equal(got[n], want[n]) for n in size), moved
