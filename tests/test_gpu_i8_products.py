"""The 8-bit integer quantizers and the dense and grouped integer products on the GPU. The products and the quantizer of plain rows are
defined to the bit (i8_ref), and held to that."""
import ctypes as C

import numpy as np
import pytest

import fp8_ref as R
import i8_ref as Q
import vbmoe as vb
from test_gpu_fp8_products import glu_values
from test_i8_products import cases

pytestmark = pytest.mark.gpu
F32, F16, BF16, I8 = 0, 1, 30, 24
TYPES = [F32, F16, BF16]


def sync(stream=None):
    vb.call("vbm_stream_synchronize", stream)


# ------------------------------------------------------------------------------------- quantizers
def quantize(type_id, x, stride=None, offset=0):
    rows, k = x.shape
    stride = stride or k
    raw, _ = R.store_as(type_id, x)
    host = np.zeros(offset + rows * stride, raw.dtype)
    host[offset:].reshape(rows, stride)[:, :k] = raw
    dx, dc, ds = vb.DeviceBuffer.from_array(host), R.filled(rows * k + 64), R.filled(4 * rows + 64)
    vb.call("vbm_quantize_i8", type_id, dx.ptr + offset * R.SIZE[type_id], rows, k, stride, dc.ptr, ds.ptr, None)
    sync()
    codes, scales = dc.download(np.uint8, (dc.nbytes,)), ds.download(np.uint8, (ds.nbytes,))
    assert (codes[rows * k:] == R.FILL).all() and (scales[4 * rows:] == R.FILL).all()
    return codes[:rows * k].view(np.int8).reshape(rows, k), scales[:4 * rows].view(np.float32)


def same(got, want):
    (codes, scales), (c, s) = got, want
    assert np.array_equal(scales, s, equal_nan=True), np.argwhere(scales != s)[:4]
    assert np.array_equal(codes, c), (int((codes != c).sum()), np.argwhere(codes != c)[:4])


@pytest.mark.parametrize("type_id", TYPES)
@pytest.mark.parametrize("rows,k,stride,offset", [(1, 16, None, 0), (1, 2880, None, 0), (5, 512, None, 0), (7, 528, None, 0), (3, 2048, 2064, 0), (37, 2064, 2069, 1),
                                                  (9, 4096, None, 0), (6, 4112, 4200, 8), (4, 8192, None, 0), (3, 8208, None, 0), (2, 16384, None, 0),
                                                  (2, 16400, None, 0), (2, 65536, 65537, 3), (1000, 208, None, 0), (5000, 96, 97, 0),
                                                  (513, 2304, None, 0), (700, 4400, 4401, 0)])
def test_quantize(gpu, type_id, rows, k, stride, offset):
    rng = np.random.default_rng(rows * 7 + k)
    x = (rng.standard_normal((rows, k)) * np.exp2(rng.integers(-6, 6, (rows, 1)))).astype(np.float32)
    x[:, rng.integers(0, k)] *= 20
    same(quantize(type_id, x, stride, offset), Q.quantize(R.store_as(type_id, x)[1]))


@pytest.mark.parametrize("type_id", TYPES)
def test_quantize_edges(gpu, type_id):
    """Zeros, ties, the types' largest and smallest values, and rows that hold something that is no number."""
    rng = np.random.default_rng(2)
    k = 2576
    x = rng.standard_normal((12, k)).astype(np.float32)
    big = {F32: 3.4e38, F16: 65504.0, BF16: 3.3e38}[type_id]
    x[0] = 0.0
    x[1] = -0.0
    x[2] = rng.integers(-254, 255, k) / 2                                # ties of whole codes
    x[2, 7] = 127.0
    x[3, 5] = np.nan
    x[4, k - 1] = -np.inf
    x[5] *= np.float32(1e-30)
    x[6] *= np.float32(1e-38)
    x[7] = big * np.sign(x[7])
    x[8, 0] = big
    x[9, 1:] = 0.0
    x[10, :] = np.float32(2.0) ** rng.integers(-20, 10, k)
    got = quantize(type_id, x)
    same(got, Q.quantize(R.store_as(type_id, x)[1]))
    assert np.array_equal(np.isnan(got[1]), np.isin(np.arange(12), (3, 4))) and (got[0][3:5] == 0).all()


@pytest.mark.parametrize("type_id", TYPES)
@pytest.mark.parametrize("act", [0, 1])
@pytest.mark.parametrize("rows,width,extra,offset,size", [(1, 16, 0, 0, 1), (8, 768, 0, 0, 3), (33, 2880, 0, 0, 10), (5, 208, 5, 1, 60), (3, 9008, 0, 0, 2)])
def test_glu_quantize(gpu, type_id, act, rows, width, extra, offset, size):
    """The value's relative error: the argument of the exponential is rounded (2^-24 of it, a relative error of |argument| 2^-24 in the
    result), and eight more roundings follow. The scale is off by that; a code by half a step and 127 times twice that."""
    rng = np.random.default_rng(width + act)
    alpha, limit, stride = 1.702, 7.0, 2 * width + extra
    x = rng.standard_normal((rows, stride)).astype(np.float32) * size
    x[0, :8] = 0.0
    if size >= 10:
        x[0, 8], x[0, 9] = -200.0, -95.0                                 # exponentials past the fp32 range
    raw, v = R.store_as(type_id, x)
    host = np.zeros(offset + raw.size, raw.dtype)
    host[offset:] = raw.reshape(-1)
    dx, es = vb.DeviceBuffer.from_array(host), R.SIZE[type_id]
    dc, ds = R.filled(rows * width + 64), R.filled(4 * rows + 64)
    vb.call("vbm_glu_quantize_i8", act, type_id, dx.ptr + offset * es, dx.ptr + (offset + width) * es, rows, width, stride, stride,
            alpha, limit, dc.ptr, ds.ptr, None)
    sync()
    assert (dc.download(np.uint8, (dc.nbytes,))[rows * width:] == R.FILL).all()
    codes, scales = dc.download(np.int8, (rows, width)), ds.download(np.float32, (rows,)).astype(np.float64)
    h = glu_values(act, v[:, :width], v[:, width:2 * width], float(np.float32(alpha)), limit)
    a = np.maximum(np.abs(h).max(axis=1), float(R.LEAST))
    rel = (np.abs(v[:, :width]).max() * alpha + 8) * 2.0 ** -24
    assert (np.abs(scales - a / 127) <= rel * a / 127).all()
    assert (np.abs(codes - h * (127 / a)[:, None]) <= 0.5 + 2 * rel * 127 + 127 * 2.0 ** -23).all()


def test_glu_quantize_marks_rows_without_a_scale(gpu):
    width = 256
    x = np.ones((3, 2 * width), np.float32)
    x[1, 3] = np.nan
    x[2, width + 200] = np.inf
    dx, dc, ds = vb.DeviceBuffer.from_array(x), vb.DeviceBuffer(3 * width), vb.DeviceBuffer(12)
    vb.call("vbm_glu_quantize_i8", 0, F32, dx.ptr, dx.ptr + 4 * width, 3, width, 2 * width, 2 * width, 1.702, 7.0, dc.ptr, ds.ptr, None)
    sync()
    scales, codes = ds.download(np.float32, (3,)), dc.download(np.int8, (3, width))
    assert np.array_equal(np.isnan(scales), [False, True, True])
    assert (codes[1:] == 0).all() and (codes[0] == 127).all()


# ---------------------------------------------------------------------------------- dense product
@pytest.mark.parametrize("dst_type", TYPES)
@pytest.mark.parametrize("tokens,rows,k,bias", [(1, 64, 128, False), (1, 300, 2880, True), (2, 1, 16, True), (15, 129, 48, False), (16, 15, 144, False),
                                                (17, 100, 336, True), (40, 130, 2048, False), (65, 257, 720, True), (130, 515, 400, False),
                                                (300, 384, 1040, True), (2085, 6164, 144, True), (1000, 2000, 272, False),
                                                (3, 70, 8720, True), (9, 33, 8832, False), (300, 130, 8720, True), (2500, 4100, 2320, False)])
def test_dense_product(gpu, dst_type, tokens, rows, k, bias):
    rng = np.random.default_rng(tokens * 31 + rows)
    m, x = Q.Matrix(rng, 1, rows, k, bias), Q.Tokens(rng, tokens, k)
    dst = R.filled((tokens + 1) * rows * R.SIZE[dst_type])
    vb.call("vbm_mul_mat_i8", m.desc, x.data.ptr, x.scales.ptr, tokens, dst_type, dst.ptr, None)
    sync()
    got = R.load_as(dst_type, dst, (tokens + 1, rows))
    Q.check(dst_type, got, *Q.grouped_want(m, x, tokens, [0, tokens], tokens, tokens + 1, dst_type))


@pytest.mark.parametrize("tokens", [1, 33, 300])
def test_the_largest_sums(gpu, tokens):
    """-128 times -128 over the deepest rows: 131056 * 2^14 is just below 2^31."""
    rows, k = 65, 131056
    x = np.full((tokens, k), -128, np.int8)
    w = np.full((1, rows, k), -128, np.int8)
    w[0, 1::2] = 127
    one = np.ones(max(rows, tokens), np.float32)
    d = [vb.DeviceBuffer.from_array(a) for a in (w, x, one)]
    dst = vb.DeviceBuffer(tokens * rows * 4)
    vb.call("vbm_mul_mat_i8", vb.Weights(I8, d[0].ptr, d[2].ptr, None, 1, rows, k), d[1].ptr, d[2].ptr, tokens, F32, dst.ptr, None)
    sync()
    want = np.where(np.arange(rows) % 2, np.float32(-128 * 127 * k), np.float32(128 * 128 * k))
    assert np.array_equal(dst.download(np.float32, (tokens, rows)), np.broadcast_to(want, (tokens, rows)))


@pytest.mark.parametrize("dst_type,offset", [(F32, 4), (F32, 8), (F16, 2), (BF16, 6), (BF16, 8)])
@pytest.mark.parametrize("tokens,rows", [(2, 64), (30, 72), (333, 256)])
def test_outputs_that_are_aligned_to_their_type_only(gpu, dst_type, offset, tokens, rows):
    rng = np.random.default_rng(offset + tokens)
    m, x = Q.Matrix(rng, 1, rows, 208, True), Q.Tokens(rng, tokens, 208)
    size = tokens * rows * R.SIZE[dst_type]
    dst = R.filled(16 + size + 64)
    vb.call("vbm_mul_mat_i8", m.desc, x.data.ptr, x.scales.ptr, tokens, dst_type, dst.ptr + offset, None)
    sync()
    raw = dst.download(np.uint8, (dst.nbytes,))
    assert (raw[:offset] == R.FILL).all() and (raw[offset + size:] == R.FILL).all()
    out = raw[offset:offset + size].copy()
    got = {F32: lambda: out.view(np.float32), F16: lambda: out.view(np.float16), BF16: lambda: R.bf16_values(out.view(np.uint16))}[dst_type]()
    Q.check(dst_type, got.astype(np.float64).reshape(tokens, rows), *Q.grouped_want(m, x, tokens, [0, tokens], tokens, tokens, dst_type))


def test_scales_that_are_not_numbers(gpu):
    """A NaN token scale (a row that had no scale), an infinite and a NaN weight scale reach the outputs that read them, and no others."""
    rng = np.random.default_rng(5)
    for tokens in (4, 100, 400):
        m, x = Q.Matrix(rng, 1, 160, 400), Q.Tokens(rng, tokens, 400)
        ws, bs = m.scale_values[0].copy(), x.scale_values.copy()
        ws[7], ws[9], bs[1] = np.nan, np.inf, np.nan
        d = [vb.DeviceBuffer.from_array(a) for a in (ws, bs)]
        dst = vb.DeviceBuffer(tokens * 160 * 4)
        vb.call("vbm_mul_mat_i8", vb.Weights(I8, m.data.ptr, d[0].ptr, None, 1, 160, 400), x.data.ptr, d[1].ptr, tokens, F32, dst.ptr, None)
        sync()
        want = np.ones((tokens, 160), bool)
        want[:, [7, 9]] = False
        want[1] = False
        assert np.array_equal(np.isfinite(dst.download(np.float32, (tokens, 160))), want)


# -------------------------------------------------------------------------------- grouped product
@pytest.mark.parametrize("dst_type", [F32, BF16])
@pytest.mark.parametrize("counts", [[0, 1, 0], [0, 0, 5, 0, 17, 0], [16, 15, 33, 1, 64, 63, 65], [0, 0, 150, 0], [300, 0, 129, 257, 31], [0, 0, 0]])
@pytest.mark.parametrize("gather", [True, False])
def test_grouped_product(gpu, dst_type, counts, gather):
    rng = np.random.default_rng(len(counts) * 7 + gather)
    used, rows, k, top_k = sum(counts), 200, 336, 4
    n_rows = used + 3
    m = Q.Matrix(rng, len(counts), rows, k, bias=gather)
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    place = rng.permutation(n_rows).astype(np.int32)
    n_b = -(-n_rows // top_k) if gather else n_rows
    x = Q.Tokens(rng, n_b, k)
    kw = dict(b_rows=place, b_div=top_k) if gather else dict(dst_rows=place)
    got = R.grouped(m, x, n_b, offsets, n_rows, dst_type, n_rows, **kw)
    Q.check(dst_type, got, *Q.grouped_want(m, x, n_b, offsets, n_rows, n_rows, dst_type, **kw))


CASES = list(cases())


@pytest.mark.parametrize("dst_type", [F32, BF16])
@pytest.mark.parametrize("name,groups,mean,rows,k", CASES, ids=[c[0].replace(" ", "_") for c in CASES])
def test_every_kernel(gpu, name, groups, mean, rows, k, dst_type):
    """Each kernel with rows out of range, offsets past the end and scattered outputs; and again with other work in between: the same bits."""
    rng = np.random.default_rng(len(name) * 100 + dst_type)
    n_rows, n_b = groups * mean, 301
    counts = rng.multinomial(n_rows - 2, rng.dirichlet(np.full(groups, 4.0)))
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    offsets[-1] += 50
    m, x = Q.Matrix(rng, groups, rows, k, bias=True, distinct=min(3, groups)), Q.Tokens(rng, n_b, k)
    b_rows, dst_rows = rng.integers(0, 2 * n_b, n_rows).astype(np.int32), rng.permutation(n_rows).astype(np.int32)
    pick = rng.permutation(n_rows)
    b_rows[pick[:3]] = [-1, 2 * n_b, 2 ** 31 - 1]
    dst_rows[pick[3:5]] = [-1, n_rows]
    kw = dict(b_rows=b_rows, b_div=2, dst_rows=dst_rows)
    want = Q.grouped_want(m, x, n_b, offsets, n_rows, n_rows, dst_type, **kw)
    for _ in range(2):
        Q.check(dst_type, R.grouped(m, x, n_b, offsets, n_rows, dst_type, n_rows, **kw), *want)
        quantize(F32, np.ones((64, 4096), np.float32))


# --------------------------------------------------------------------------- together, in a layer
class Layer:
    """A residual stream's next rows through a layer of integer experts, as the calls are meant to be chained: residual and norm, routing by
    the normed rows, the experts on their codes."""

    def __init__(self, rng, T, H, I, E, K, act):
        self.T, self.H, self.I, self.E, self.K, self.act = T, H, I, E, K, act
        self.gu, self.dn = Q.Matrix(rng, E, 2 * I, H, True), Q.Matrix(rng, E, H, I, True)
        self.x, self.residual = (rng.standard_normal((T, H)).astype(np.float32) for _ in range(2))
        self.weight = (rng.random(H) + 0.5).astype(np.float32)
        self.router = (rng.standard_normal((E, H)) / np.sqrt(H)).astype(np.float32)
        n = T * K
        self.b = {name: vb.DeviceBuffer(size) for name, size in dict(
            sum=4 * T * H, y=4 * T * H, logits=4 * T * E, ids=4 * n, weights=4 * n, counts=4 * E, offsets=4 * (E + 1), rows=4 * n, xc=T * H,
            xs=4 * T, gu=2 * n * 2 * I, hc=n * I, hs=4 * n, ye=4 * n * H, out=4 * T * H).items()}
        for name in ("x", "residual", "weight", "router"):
            self.b[name] = vb.DeviceBuffer.from_array(getattr(self, name))

    def enqueue(self, s):
        T, H, I, E, K, n = self.T, self.H, self.I, self.E, self.K, self.T * self.K
        p = {name: buf.ptr for name, buf in self.b.items()}
        vb.call("vbm_add_rms_norm_quantize", F32, p["x"], H, p["residual"], p["sum"], H, p["weight"], T, H, 1e-6, F32, p["y"], I8, p["xc"], p["xs"], s)
        vb.call("vbm_router_topk_softmax", p["router"], None, p["y"], H, p["logits"], E, T, K, p["ids"], p["weights"], s)
        vb.call("vbm_group_by_expert", p["ids"], K, T, K, E, p["counts"], p["offsets"], p["rows"], None, s)
        vb.call("vbm_grouped_mul_mat", self.gu.desc, p["xc"], p["xs"], T, p["rows"], K, p["offsets"], n, None, n, BF16, p["gu"], s)
        vb.call("vbm_glu_quantize_i8", self.act, BF16, p["gu"], p["gu"] + 2 * I, n, I, 2 * I, 2 * I, 1.702, 7.0, p["hc"], p["hs"], s)
        vb.call("vbm_grouped_mul_mat", self.dn.desc, p["hc"], p["hs"], n, None, 1, p["offsets"], n, p["rows"], n, F32, p["ye"], s)
        vb.call("vbm_weighted_combine", p["ye"], p["weights"], H, K, T, p["out"], s)


@pytest.mark.parametrize("T,H,I,E,K,act", [(1, 256, 192, 8, 2, 0), (5, 2880, 336, 8, 4, 1), (200, 512, 400, 8, 4, 1)])
def test_layer_of_integer_experts(gpu, T, H, I, E, K, act):
    """The chain against float64, step by step on the codes that the steps before it left: each rounding is then counted once. An output is
    held to the roundings of bf16 gate and up values (2^-8 each) and of the integer activations (half a code each) through |down|."""
    rng = np.random.default_rng(T + H)
    s = C.c_void_p()
    vb.call("vbm_stream_create", C.byref(s))
    L = Layer(rng, T, H, I, E, K, act)
    L.enqueue(s.value)
    sync(s.value)
    total = (L.x + L.residual).astype(np.float32)
    assert np.array_equal(L.b["sum"].download(np.float32, (T, H)), total)
    v = total.astype(np.float64)
    y = v / np.sqrt((v * v).mean(axis=1, keepdims=True) + float(np.float32(1e-6))) * L.weight
    assert np.abs(L.b["y"].download(np.float32, (T, H)) - y).max() <= 64 * 2.0 ** -24 * np.abs(y).max()
    xc, xs = L.b["xc"].download(np.int8, (T, H)), L.b["xs"].download(np.float32, (T,))
    a = np.abs(y).max(axis=1)
    assert np.abs(xc - y * (127 / a)[:, None]).max() <= 0.5 + 127 * 64 * 2.0 ** -23
    xq = xc * xs.astype(np.float64)[:, None]
    ids, w = L.b["ids"].download(np.int32, (T, K)), L.b["weights"].download(np.float32, (T, K)).astype(np.float64)
    logits = y @ L.router.astype(np.float64).T
    assert (np.sort(np.take_along_axis(logits, ids, 1), axis=1) >= np.sort(logits, axis=1)[:, -K:] - 1e-4).all()
    got = L.b["out"].download(np.float32, (T, H)).astype(np.float64)
    want, bound = np.zeros((T, H)), np.zeros((T, H))
    values = lambda m, e: m.codes[e] * m.scale_values[e].astype(np.float64)[:, None]  # noqa: E731
    for t in range(T):
        for j, e in enumerate(ids[t]):
            g = values(L.gu, e) @ xq[t] + L.gu.bias_values[e]
            h = glu_values(act, g[:I], g[I:], 1.702, 7.0)
            d = values(L.dn, e)
            want[t] += w[t, j] * (d @ h + L.dn.bias_values[e])
            # (|d glu / d gate| <= 1.13 (|up| + 1), |d glu / d up| <= |gate|)
            dh = 2.0 ** -8 * (1.2 * np.abs(g[:I]) * (np.abs(g[I:]) + 1) + np.abs(g[:I]) * np.abs(g[I:])) * 1.01
            dh = dh + (np.abs(h) + dh).max() / 254 * 1.01
            bound[t] += w[t, j] * (np.abs(d) @ dh + 1e-4)
    err = np.abs(got - want)
    assert (err <= bound).all(), float((err / bound).max())
    print(f"[integer layer T={T}] rel {np.linalg.norm(got - want) / np.linalg.norm(want):.4f}", flush=True)
    vb.call("vbm_stream_destroy", s.value)


def test_captured_layer_replays_on_new_inputs(gpu):
    """One graph of the chain, replayed with new rows between eager calls on another stream: the eager results' bits."""
    rng = np.random.default_rng(77)
    T, H, I, E, K = 40, 512, 256, 8, 2
    s1, s2, graph = C.c_void_p(), C.c_void_p(), C.c_void_p()
    vb.call("vbm_stream_create", C.byref(s1))
    vb.call("vbm_stream_create", C.byref(s2))
    L = Layer(rng, T, H, I, E, K, 1)
    L.enqueue(s1.value)                                 # (the grouping's scratch is allocated by a first call)
    sync(s1.value)
    vb.call("vbm_graph_begin_capture", s1.value)
    L.enqueue(s1.value)
    vb.call("vbm_graph_end_capture", s1.value, C.byref(graph))
    for step in range(4):
        L.b["x"].upload(rng.standard_normal((T, H)).astype(np.float32), s1.value)
        L.enqueue(s2.value)
        sync(s2.value)
        want = L.b["out"].download(np.uint32, (T, H))
        vb.call("vbm_memset", L.b["out"].ptr, 0, L.b["out"].nbytes, s1.value)
        sync(s1.value)
        vb.call("vbm_graph_launch", graph.value, s1.value)
        sync(s1.value)
        assert np.array_equal(L.b["out"].download(np.uint32, (T, H)), want), step
    vb.call("vbm_graph_destroy", graph.value)
    for s in (s1, s2):
        vb.call("vbm_stream_destroy", s.value)


def test_two_streams_at_once(gpu):
    """The same calls in flight on two streams give what they give alone."""
    rng = np.random.default_rng(78)
    streams, layers = [C.c_void_p(), C.c_void_p()], []
    for s in streams:
        vb.call("vbm_stream_create", C.byref(s))
        layers.append(Layer(rng, 64, 512, 256, 8, 2, 0))
    alone = []
    for s, layer in zip(streams, layers):
        layer.enqueue(s.value)
        sync(s.value)
        alone.append(layer.b["out"].download(np.uint32, (64, 512)))
    for _ in range(3):
        for _ in range(4):
            for s, layer in zip(streams, layers):
                layer.enqueue(s.value)
        for s in streams:
            sync(s.value)
        for want, layer in zip(alone, layers):
            assert np.array_equal(layer.b["out"].download(np.uint32, (64, 512)), want)
    for s in streams:
        vb.call("vbm_stream_destroy", s.value)
