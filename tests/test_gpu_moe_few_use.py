"""vbm_moe_few_forward as a program uses it: a padded batch, and two captured layers of different sizes that share one workspace."""
import ctypes as C

import numpy as np
import pytest

import vbmoe as vb
from test_gpu_moe_few import F32, BF16, F8, I8, KINDS, Layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("x_type", [F32, BF16])
def test_padding_tokens_are_not_read(gpu, kind, x_type):
    """Tokens without experts (all ids -1) hold anything, NaN here: they come out as zeros, and the others as without them."""
    L = Layer(kind, 6, 272, 96, 3, 1, True, seed=21)
    T, pad = 11, [0, 4, 5, 10]
    raw, _ = L.tokens(T, x_type)
    ids = np.argsort(L.rng.random((T, 6)), axis=1)[:, :3].astype(np.int32)
    weights = L.rng.random((T, 3)).astype(np.float32)
    ids[pad] = -1
    weights[pad] = np.nan
    want, _, _ = L.run(T, x_type, raw, ids=ids, weights=weights)
    raw[pad] = 0x7FC0 if x_type == BF16 else np.nan
    got, _, _ = L.run(T, x_type, raw, ids=ids, weights=weights)
    assert np.array_equal(got, want) and (got[pad] == 0).all() and np.isfinite(got).all()


def test_two_captured_layers_share_a_workspace(gpu):
    """Graphs of an FP8 layer for six tokens and an integer one for three, replayed in turn on one stream and out of turn: the eager results' bits each time."""
    layers = [(Layer(F8, 8, 400, 272, 4, 1, True, seed=22), 6), (Layer(I8, 12, 144, 1040, 2, 0, True, seed=23), 3)]
    size = max(L.workspace(T) for L, T in layers)
    s, ws, own = C.c_void_p(), vb.DeviceBuffer(size), vb.DeviceBuffer(size)
    vb.call("vbm_stream_create", C.byref(s))
    calls = []
    for L, T in layers:
        d = {"x": vb.DeviceBuffer(4 * T * L.H), "logits": vb.DeviceBuffer(4 * T * L.E), "out": vb.DeviceBuffer(4 * T * L.H)}
        graph = C.c_void_p()

        def enqueue(stream, space, L=L, T=T, d=d):
            vb.call("vbm_moe_few_forward", L.desc, F32, d["x"].ptr, d["logits"].ptr, None, None, T, F32, d["out"].ptr, space.ptr, size, stream)

        vb.call("vbm_graph_begin_capture", s.value)
        enqueue(s.value, ws)
        vb.call("vbm_graph_end_capture", s.value, C.byref(graph))
        calls.append((L, T, d, graph, enqueue))
    for order in ([0, 1], [1, 0, 1], [0, 0, 1], [1, 1, 0]):
        want = []
        for L, T, d, _, enqueue in calls:
            d["x"].upload(L.rng.standard_normal((T, L.H)).astype(np.float32), s.value)
            d["logits"].upload(L.rng.standard_normal((T, L.E)).astype(np.float32), s.value)
            enqueue(None, own)
            vb.call("vbm_stream_synchronize", None)
            want.append(d["out"].download(np.uint32, (T, L.H)))
            vb.call("vbm_memset", d["out"].ptr, 0, d["out"].nbytes, None)
            vb.call("vbm_stream_synchronize", None)
        for i in order:
            vb.call("vbm_graph_launch", calls[i][3].value, s.value)
        vb.call("vbm_stream_synchronize", s.value)
        for (L, T, d, *_), w in zip(calls, want):
            assert np.array_equal(d["out"].download(np.uint32, (T, L.H)), w), order
    for *_, graph, _ in calls:
        vb.call("vbm_graph_destroy", graph.value)
    vb.call("vbm_stream_destroy", s.value)
