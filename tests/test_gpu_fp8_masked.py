"""The chain of an FP8 layer where some routes are masked: y is zeroed first, in the captured graph too."""
import ctypes as C

import numpy as np
import pytest

import fp8_ref as R
import vbmoe as vb

pytestmark = pytest.mark.gpu
F32, BF16, F8 = 0, 30, 256


def streams_of(n):
    s = [C.c_void_p() for _ in range(n)]
    for x in s:
        vb.call("vbm_stream_create", C.byref(x))
    return s


@pytest.mark.parametrize("offset,nbytes", [(0, 1), (3, 5), (15, 1), (15, 17), (0, 64), (1, 4096 + 7), (8, 3_000_001), (0, 1 << 26)])
def test_captured_memset_fills_what_it_says(gpu, offset, nbytes):
    """Replayed three times, over other contents each time."""
    (s,) = streams_of(1)
    buf, graph = R.filled(offset + nbytes + 32), C.c_void_p()
    vb.call("vbm_graph_begin_capture", s.value)
    vb.call("vbm_memset", buf.ptr + offset, 0x1C3, nbytes, s.value)       # (the low byte counts, as in memset)
    vb.call("vbm_graph_end_capture", s.value, C.byref(graph))
    for _ in range(3):
        vb.call("vbm_memset", buf.ptr, R.FILL, buf.nbytes, s.value)
        vb.call("vbm_graph_launch", graph.value, s.value)
        vb.call("vbm_stream_synchronize", s.value)
        got = buf.download(np.uint8, (buf.nbytes,))
        assert (got[offset:offset + nbytes] == 0xC3).all()
        assert (got[:offset] == R.FILL).all() and (got[offset + nbytes:] == R.FILL).all()
    vb.call("vbm_graph_destroy", graph.value)
    vb.call("vbm_stream_destroy", s.value)


@pytest.mark.parametrize("T", [3, 90])
def test_masked_routes_through_the_down_product_and_combine(gpu, T):
    """Captured once with y's zeroing in it and replayed over other masks: the eager bits, and the sums of the routes that are left. Each
    output is off by the product's bound and one rounding a rank, each of at most the magnitudes' sum."""
    rng = np.random.default_rng(T)
    H, I, E, K = 200, 336, 8, 3
    n = T * K
    dn, h = R.Matrix(F8, rng, E, H, I, bias=True), R.Tokens(F8, rng, n, I)
    ids, weights = vb.DeviceBuffer(4 * n), vb.DeviceBuffer(4 * n)
    counts, offsets, rows, y, out = (vb.DeviceBuffer(4 * m) for m in (E, E + 1, n, n * H, T * H))

    def enqueue(s):
        vb.call("vbm_group_by_expert", ids.ptr, K, T, K, E, counts.ptr, offsets.ptr, rows.ptr, None, s)
        vb.call("vbm_memset", y.ptr, 0, y.nbytes, s)
        vb.call("vbm_grouped_mul_mat", dn.desc, h.data.ptr, h.scales.ptr, n, None, 1, offsets.ptr, n, rows.ptr, n, F32, y.ptr, s)
        vb.call("vbm_weighted_combine", y.ptr, weights.ptr, H, K, T, out.ptr, s)

    s1, s2 = streams_of(2)
    ids.upload(np.zeros((T, K), np.int32), s1.value)
    weights.upload(np.zeros((T, K), np.float32), s1.value)
    enqueue(s1.value)                                   # (the grouping's scratch is allocated by a first call)
    vb.call("vbm_stream_synchronize", s1.value)
    graph = C.c_void_p()
    vb.call("vbm_graph_begin_capture", s1.value)
    enqueue(s1.value)
    vb.call("vbm_graph_end_capture", s1.value, C.byref(graph))
    for step in range(4):
        route = np.stack([rng.permutation(E)[:K] for _ in range(T)]).astype(np.int32)
        w = rng.random((T, K)).astype(np.float32)
        masked = rng.random((T, K)) < (0.3, 1.0, 0.0, 0.6)[step]
        route[masked], w[masked] = -1, 0.0
        ids.upload(route, s1.value)
        weights.upload(w, s1.value)
        results = []
        for launch, s in ((lambda: enqueue(s2.value), s2.value), (lambda: vb.call("vbm_graph_launch", graph.value, s1.value), s1.value)):
            vb.call("vbm_memset", y.ptr, 0xFF, y.nbytes, s)                # NaN
            launch()
            vb.call("vbm_stream_synchronize", s)
            results.append(out.download(np.float32, (T, H)))
        assert np.array_equal(results[0].view(np.uint32), results[1].view(np.uint32)), step
        want, bound = np.zeros((T, H)), np.zeros((T, H))
        order = np.argsort(np.where(masked, E, route).reshape(-1), kind="stable")
        place = np.empty(n, np.int64)
        place[order] = np.arange(n)                     # (token, rank) -> grouped row, whose tokens the down product reads
        for t in range(T):
            for j in range(K):
                if masked[t, j]:
                    continue
                x = h.values[place[t * K + j]]
                v = dn.values[route[t, j]] @ x + dn.bias_values[route[t, j]]
                size = np.abs(dn.values[route[t, j]]) @ np.abs(x) + np.abs(dn.bias_values[route[t, j]])
                want[t] += w[t, j] * v
                bound[t] += w[t, j] * (R.sum_bound(F8, F32, I, v, size) + 2 * K * 2.0 ** -24 * size)
        assert (np.abs(results[1] - want) <= bound).all(), step
    vb.call("vbm_graph_destroy", graph.value)
    for s in (s1, s2):
        vb.call("vbm_stream_destroy", s.value)
