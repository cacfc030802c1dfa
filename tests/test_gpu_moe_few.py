"""vbm_moe_few_forward on the GPU against float64."""
import ctypes as C

import numpy as np
import pytest

import fp8_ref as R
import i8_ref as Q
import vbmoe as vb

pytestmark = pytest.mark.gpu
F32, F16, BF16, F8, I8 = 0, 1, 30, 256, 24
ALPHA, LIMIT = 1.702, 7.0


def matrix(kind, rng, groups, rows, k, bias):
    if kind == I8:
        m = Q.Matrix(rng, groups, rows, k, bias)
        m.scale_values = (m.scale_values / np.sqrt(k)).astype(np.float32) * np.float32(15)
        m.scales.upload(m.scale_values)
        m.values = m.codes * m.scale_values.astype(np.float64)[:, :, None]
        return m
    return R.Matrix(kind, rng, groups, rows, k, bias)


class Layer:
    def __init__(self, kind, E, H, I, K, act, bias, seed):
        self.rng = np.random.default_rng(seed)
        self.E, self.H, self.I, self.K, self.act = E, H, I, K, act
        self.gu, self.dn = matrix(kind, self.rng, E, 2 * I, H, bias), matrix(kind, self.rng, E, H, I, bias)
        self.desc = vb.MoeFewDesc(self.gu.desc, self.dn.desc, K, act, ALPHA, LIMIT)

    def workspace(self, T):
        size = C.c_size_t()
        vb.call("vbm_moe_few_workspace", self.desc, T, size)
        return size.value

    def tokens(self, T, x_type):
        return R.store_as(x_type, self.rng.standard_normal((T, self.H)))

    def run(self, T, x_type, raw, logits=None, ids=None, weights=None, out_type=F32, returns=True, offset=0):
        """(out, ids, weights); nothing behind the buffers is written."""
        n, size = T * self.K, self.workspace(T)
        up = lambda a, t: vb.DeviceBuffer.from_array(np.ascontiguousarray(a, t)) if a is not None else None  # noqa: E731
        dx, dl = vb.DeviceBuffer.from_array(raw), up(logits, np.float32)
        di, dw = (up(ids, np.int32), up(weights, np.float32)) if logits is None else (R.filled(4 * n + 64), R.filled(4 * n + 64)) if returns else (None, None)
        es = R.SIZE[out_type]
        ws, out = R.filled(size + 256), R.filled(offset * es + T * self.H * es + 64)
        vb.call("vbm_moe_few_forward", self.desc, x_type, dx.ptr, vb.ptr(dl), vb.ptr(di), vb.ptr(dw), T, out_type, out.ptr + offset * es, ws.ptr, size, None)
        vb.call("vbm_stream_synchronize", None)
        assert (ws.download(np.uint8, (ws.nbytes,))[size:] == R.FILL).all()
        b = out.download(np.uint8, (out.nbytes,))
        assert (b[:offset * es] == R.FILL).all() and (b[-64:] == R.FILL).all()
        if logits is not None and returns:
            assert (di.download(np.uint8, (di.nbytes,))[4 * n:] == R.FILL).all() and (dw.download(np.uint8, (dw.nbytes,))[4 * n:] == R.FILL).all()
        v = np.ascontiguousarray(b[offset * es:-64])
        v = {F32: lambda: v.view(np.float32), F16: lambda: v.view(np.float16), BF16: lambda: R.bf16_values(v.view(np.uint16))}[out_type]()
        got = (di.download(np.int32, (T, self.K)), dw.download(np.float32, (T, self.K))) if di is not None else (None, None)
        return v.astype(np.float64).reshape(T, self.H), *got

    def want(self, x, ids, weights, out_type):
        """(values, bounds). The products are exact in fp32, up to six terms a weight's product; they, the FP8 blocks' scaled sums, scales and biases are added
        in fp32, each addition off by at most a step (2^-23) of a partial sum no larger than the terms' magnitudes. The GLU passes gate's and up's
        errors on (|d / d gate| <= 1.1 (|up| + 1), |d / d up| <= |gate|) and adds its own (the exponential's rounded argument, and eight
        more roundings); the ranks' sum is one rounding a product and one an addition."""
        T = x.shape[0]
        y, b = np.zeros((T, self.H)), np.zeros((T, self.H))
        step = lambda k: (6 * k + 2 * -(-k // 128) + 16) * 2.0 ** -23  # noqa: E731
        for t in range(T):
            for j, e in enumerate(ids[t]):
                if e == -1:
                    continue
                if not 0 <= e < self.E:
                    y[t] = np.nan
                    continue
                w1, w2 = self.gu.values[e], self.dn.values[e]
                g, dg = w1 @ x[t], step(self.H) * (np.abs(w1) @ np.abs(x[t]))
                if self.gu.bias_values is not None:
                    g, dg = g + self.gu.bias_values[e], dg + step(self.H) * np.abs(self.gu.bias_values[e])
                gate, up, dgate, dup = g[:self.I], g[self.I:], dg[:self.I], dg[self.I:]
                with np.errstate(over="ignore"):
                    if self.act:
                        gc, uc = np.minimum(gate, LIMIT), np.clip(up, -LIMIT, LIMIT)
                        h = gc / (1 + np.exp(-float(np.float32(ALPHA)) * gc)) * (uc + 1)
                    else:
                        h = gate / (1 + np.exp(-gate)) * up
                dh = 1.1 * (np.abs(up) + 1) * dgate + np.abs(gate) * dup + (ALPHA * np.abs(gate) + 8) * 2.0 ** -24 * np.abs(h)
                v, dv = w2 @ h, step(self.I) * (np.abs(w2) @ np.abs(h)) + np.abs(w2) @ dh
                if self.dn.bias_values is not None:
                    v, dv = v + self.dn.bias_values[e], dv + step(self.I) * np.abs(self.dn.bias_values[e])
                y[t] += float(weights[t, j]) * v
                b[t] += abs(float(weights[t, j])) * (dv + (self.K + 2) * 2.0 ** -24 * np.abs(v))
        return y, b + R.HALF_STEP[out_type] * (np.abs(y) + b) + R.LEAST_STEP[out_type]

    def check(self, T, x_type, out_type=F32, logits=None, ids=None, weights=None, **kw):
        raw, x = self.tokens(T, x_type)
        got, gi, gw = self.run(T, x_type, raw, logits, ids, weights, out_type, **kw)
        if logits is not None and gi is not None:
            ids, weights = routing(logits, self.K)
            assert np.array_equal(gi, ids)
            assert np.abs(gw - weights).max() <= 8 * 2.0 ** -24
            weights = gw
        elif logits is not None:
            ids, weights = routing(logits, self.K)
        y, b = self.want(x, ids, weights, out_type)
        bad = np.isnan(y).any(axis=1)
        assert np.isnan(got[bad]).all()
        err = np.abs(got - y)[~bad]
        b = b + (8 * 2.0 ** -24 * np.abs(y).max() * self.K if gi is None else 0)
        if err.size:
            print(f"worst error / bound {np.max(err / np.maximum(b[~bad], 1e-300)):.3f}", flush=True)
        assert (err <= b[~bad]).all(), np.argwhere(err > b[~bad])[:4]
        if out_type == F32 and err.size and np.abs(y[~bad]).max() > 0:
            # (errors of random signs add up as their root: no more than a handful of fp32 steps of the whole)
            assert np.linalg.norm(err) <= 4e-6 * np.linalg.norm(y[~bad])
        return got


def routing(logits, K):
    order = np.argsort(-logits, axis=1, kind="stable")[:, :K].astype(np.int32)
    z = np.take_along_axis(logits.astype(np.float64), order, 1)
    w = np.exp(z - z.max(axis=1, keepdims=True))
    return order, w / w.sum(axis=1, keepdims=True)


KINDS = [F8, I8, F16, BF16]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("x_type", [F32, F16, BF16])
@pytest.mark.parametrize("T,E,K,H,I,act,bias", [(1, 8, 2, 256, 192, 0, False), (2, 16, 4, 400, 336, 1, True), (5, 8, 4, 144, 1040, 1, True), (16, 32, 8, 272, 80, 0, True)])
def test_layer_from_logits(gpu, kind, x_type, T, E, K, H, I, act, bias):
    L = Layer(kind, E, H, I, K, act, bias, seed=T + kind)
    L.check(T, x_type, logits=L.rng.standard_normal((T, E)).astype(np.float32))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T,E,K,H,I", [(1, 12, 8, 2048, 768), (3, 6, 4, 1440, 1456), (16, 12, 4, 720, 1008), (8, 5, 5, 528, 4096), (1, 4, 1, 64, 16384 + 16),
                                         (16, 60, 8, 64, 1040), (16, 60, 8, 32, 3216)])
def test_layer_sizes(gpu, kind, T, E, K, H, I):
    """Shared and unshared depths, several row tiles a wave, rows that end inside a step."""
    L = Layer(kind, E, H, I, min(K, E), 1, True, seed=H)
    L.check(T, BF16, logits=(L.rng.standard_normal((T, E)) * 2).astype(np.float32), out_type=BF16)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("H,I", [(8, 8), (24, 72), (136, 8), (8, 200)])
def test_small_odd_eights(gpu, kind, H, I):
    L = Layer(kind, 3, H, I, 2, 0, True, seed=H + I)
    L.check(7, F32, logits=L.rng.standard_normal((7, 3)).astype(np.float32))


@pytest.mark.parametrize("kind", [F8, I8])
@pytest.mark.parametrize("H,I", [(16, 16), (48, 144), (272, 16), (16, 400)])
def test_small_odd_sixteens(gpu, kind, H, I):
    L = Layer(kind, 3, H, I, 2, 1, True, seed=H + I)
    L.check(7, F16, logits=L.rng.standard_normal((7, 3)).astype(np.float32))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case", ["one expert", "twice in a token", "nowhere", "out of range", "all pairs", "a token without experts"])
def test_given_routing(gpu, kind, case):
    """More rows of one expert than a slot holds, experts listed twice, ids of -1 and ids out of range."""
    T, E, K = {"all pairs": (16, 9, 8), "one expert": (16, 4, 1), "nowhere": (3, 4, 2)}.get(case, (6, 5, 4))
    L = Layer(kind, E, 208, 176, K, 0, True, seed=len(case))
    ids = np.argsort(L.rng.random((T, E)), axis=1)[:, :K].astype(np.int32)
    weights = L.rng.standard_normal((T, K)).astype(np.float32)
    if case == "one expert":
        ids[:] = 2
    elif case == "twice in a token":
        ids[:, 1:] = 3
    elif case == "nowhere":
        ids[:] = -1
    elif case == "out of range":
        ids[1, 2], ids[4, 0], ids[5, 3] = 5, -2, 2 ** 31 - 1
    elif case == "all pairs":
        ids[:, 3:] = 7
    else:
        ids[2], ids[0, 0], ids[5, 1:3] = -1, -1, -1
    for x_type in (F32, BF16):
        got = L.check(T, x_type, ids=ids, weights=weights)
        if case == "nowhere":
            assert (got == 0).all()
        if case == "a token without experts":
            assert (got[2] == 0).all()


@pytest.mark.parametrize("E", [1, 128, 129, 256, 257, 1024])
def test_numbers_of_experts(gpu, E):
    L = Layer(I8, E, 48, 32, min(E, 7), 1, True, seed=E)
    L.check(9, F32, logits=L.rng.standard_normal((9, E)).astype(np.float32))


def test_top_64(gpu):
    L = Layer(BF16, 70, 40, 24, 64, 0, False, seed=1)
    L.check(2, BF16, logits=L.rng.standard_normal((2, 70)).astype(np.float32))


def test_ties_and_nan_logits_route_as_the_router_does(gpu):
    L = Layer(F8, 20, 64, 64, 5, 0, False, seed=4)
    T = 6
    logits = np.round(L.rng.standard_normal((T, 20)), 0).astype(np.float32)
    logits[1, 3:9] = np.nan
    logits[2, :] = 1.0
    logits[3, 4] = np.inf
    raw, x = L.tokens(T, F32)
    _, ids, weights = L.run(T, F32, raw, logits)
    dl, di, dw = vb.DeviceBuffer.from_array(logits), vb.DeviceBuffer(4 * T * 5), vb.DeviceBuffer(4 * T * 5)
    vb.call("vbm_router_topk_softmax", None, None, None, 0, dl.ptr, 20, T, 5, di.ptr, dw.ptr, None)
    vb.call("vbm_stream_synchronize", None)
    assert np.array_equal(ids, di.download(np.int32, (T, 5)))
    assert np.array_equal(weights.view(np.uint32), dw.download(np.uint32, (T, 5)))


@pytest.mark.parametrize("out_type,offset", [(F32, 1), (F16, 1), (BF16, 3)])
def test_outputs_that_are_aligned_to_their_type_only(gpu, out_type, offset):
    L = Layer(F8, 6, 272, 96, 2, 0, True, seed=offset)
    L.check(3, F16, out_type=out_type, offset=offset, logits=L.rng.standard_normal((3, 6)).astype(np.float32))
    L.check(3, F16, out_type=out_type, returns=False, logits=L.rng.standard_normal((3, 6)).astype(np.float32))


@pytest.mark.parametrize("kind", KINDS)
def test_large_and_small_values(gpu, kind):
    """Activations and hidden values over the fp32 range, whose three terms have to cover it: tiny ones next to large ones."""
    L = Layer(kind, 4, 128, 64, 2, 0, False, seed=11)
    T = 4
    x = L.rng.standard_normal((T, 128)).astype(np.float32) * np.exp2(L.rng.integers(-40, 8, (T, 128))).astype(np.float32)
    x[1] *= np.float32(1e12)
    ids, weights = np.array([[0, 1], [2, 3], [1, 1], [3, 0]], np.int32), np.full((T, 2), 0.5, np.float32)
    got, _, _ = L.run(T, F32, x, ids=ids, weights=weights)
    y, b = L.want(x.astype(np.float64), ids, weights, F32)
    assert (np.abs(got - y) <= b).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("x_type", [F32, F16, BF16])
def test_tokens_that_are_not_numbers(gpu, kind, x_type):
    """A NaN or an infinity makes its own token's outputs NaN, and no other's, also not of a token that shares its experts."""
    L = Layer(kind, 2, 272, 80, 2, 1, True, seed=12)
    T = 5
    x = L.rng.standard_normal((T, 272))
    x[1, 271], x[3, 0] = np.nan, np.inf
    raw, v = R.store_as(x_type, x)
    ids, weights = np.tile(np.array([[0, 1]], np.int32), (T, 1)), np.full((T, 2), 0.5, np.float32)
    got, _, _ = L.run(T, x_type, raw, ids=ids, weights=weights)
    good = [0, 2, 4]
    y, b = L.want(v[good], ids[good], weights[good], F32)
    assert (np.abs(got[good] - y) <= b).all() and np.isnan(got[1]).all()


def test_it_agrees_with_the_chain_of_products(gpu):
    """The same integer layer by the chain of calls: apart from the chain's own roundings (activations to 8 bits twice: half a code of 127 each, the
    normal values' largest about four times their root mean square; gate and up to bf16) the results are one."""
    rng, T, H, I, E, K = np.random.default_rng(3), 9, 512, 400, 8, 3
    L = Layer(I8, E, H, I, K, 1, True, seed=5)
    logits = rng.standard_normal((T, E)).astype(np.float32)
    raw, x = L.tokens(T, F32)
    got, ids, weights = L.run(T, F32, raw, logits)
    n = T * K
    b = {k: vb.DeviceBuffer(v) for k, v in dict(ids=4 * n, w=4 * n, counts=4 * E, off=4 * (E + 1), rows=4 * n, xc=T * H, xs=4 * T, gu=2 * n * 2 * I, hc=n * I, hs=4 * n,
                                                y=4 * n * H, out=4 * T * H).items()}
    dx, dl = vb.DeviceBuffer.from_array(raw), vb.DeviceBuffer.from_array(logits)
    p = {k: v.ptr for k, v in b.items()}
    vb.call("vbm_router_topk_softmax", None, None, None, 0, dl.ptr, E, T, K, p["ids"], p["w"], None)
    vb.call("vbm_group_by_expert", p["ids"], K, T, K, E, p["counts"], p["off"], p["rows"], None, None)
    vb.call("vbm_quantize_i8", F32, dx.ptr, T, H, H, p["xc"], p["xs"], None)
    vb.call("vbm_grouped_mul_mat", L.gu.desc, p["xc"], p["xs"], T, p["rows"], K, p["off"], n, None, n, BF16, p["gu"], None)
    vb.call("vbm_glu_quantize_i8", 1, BF16, p["gu"], p["gu"] + 2 * I, n, I, 2 * I, 2 * I, ALPHA, LIMIT, p["hc"], p["hs"], None)
    vb.call("vbm_grouped_mul_mat", L.dn.desc, p["hc"], p["hs"], n, None, 1, p["off"], n, p["rows"], n, F32, p["y"], None)
    vb.call("vbm_weighted_combine", p["y"], p["w"], H, K, T, p["out"], None)
    vb.call("vbm_stream_synchronize", None)
    chain = b["out"].download(np.float32, (T, H)).astype(np.float64)
    assert np.array_equal(b["ids"].download(np.int32, (T, K)), ids)
    rel = np.linalg.norm(chain - got) / np.linalg.norm(got)
    print(f"chain against layer: {rel:.4f}", flush=True)
    assert rel <= 0.05


@pytest.mark.parametrize("kind,T", [(F8, 1), (BF16, 16), (I8, 4)])
def test_captured_calls_replay_on_new_inputs(gpu, kind, T):
    """A captured call replayed on new tokens and logits, between eager calls with another workspace on another stream: the eager results' bits."""
    E, K, H, I = 16, 4, 512, 272
    L = Layer(kind, E, H, I, K, 1, True, seed=T)
    s1, s2, graph = C.c_void_p(), C.c_void_p(), C.c_void_p()
    for s in (s1, s2):
        vb.call("vbm_stream_create", C.byref(s))
    size = L.workspace(T)
    dx, dl, out, other = vb.DeviceBuffer(4 * T * H), vb.DeviceBuffer(4 * T * E), vb.DeviceBuffer(4 * T * H), vb.DeviceBuffer(4 * T * H)
    ws = [vb.DeviceBuffer(size) for _ in range(2)]

    def enqueue(stream, w, o):
        vb.call("vbm_moe_few_forward", L.desc, F32, dx.ptr, dl.ptr, None, None, T, F32, o.ptr, w.ptr, size, stream)

    vb.call("vbm_graph_begin_capture", s1.value)
    enqueue(s1.value, ws[0], out)
    vb.call("vbm_graph_end_capture", s1.value, C.byref(graph))
    for step in range(4):
        dx.upload(L.rng.standard_normal((T, H)).astype(np.float32), s1.value)
        dl.upload(L.rng.standard_normal((T, E)).astype(np.float32), s1.value)
        vb.call("vbm_graph_launch", graph.value, s1.value)
        enqueue(s2.value, ws[1], other)
        for s in (s1, s2):
            vb.call("vbm_stream_synchronize", s.value)
        a, b = out.download(np.uint32, (T, H)), other.download(np.uint32, (T, H))
        assert np.array_equal(a, b) and np.isfinite(a.view(np.float32)).all(), step
    vb.call("vbm_graph_destroy", graph.value)
    for s in (s1, s2):
        vb.call("vbm_stream_destroy", s.value)


def test_out_may_be_x_and_repeated_calls_give_the_same_bits(gpu):
    L = Layer(F8, 8, 256, 128, 2, 0, False, seed=2)
    T = 8
    logits = L.rng.standard_normal((T, 8)).astype(np.float32)
    raw, _ = L.tokens(T, F32)
    want, _, _ = L.run(T, F32, raw, logits)
    for _ in range(3):
        assert np.array_equal(L.run(T, F32, raw, logits)[0], want)
    dx, dl, ws = vb.DeviceBuffer.from_array(raw), vb.DeviceBuffer.from_array(logits), vb.DeviceBuffer(L.workspace(T))
    vb.call("vbm_moe_few_forward", L.desc, F32, dx.ptr, dl.ptr, None, None, T, F32, dx.ptr, ws.ptr, ws.nbytes, None)
    vb.call("vbm_stream_synchronize", None)
    assert np.array_equal(dx.download(np.float32, (T, 256)).astype(np.float64), want)
