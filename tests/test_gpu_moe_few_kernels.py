"""vbm_moe_few_forward on the GPU: every gate_up kernel with every type of tokens, the terms that fp32 values are split into, and infinities."""
import numpy as np
import pytest

import fp8_ref as R
import i8_ref as Q
import moe_few_cases as M
import vbmoe as vb
from test_gpu_moe_few import ALPHA, LIMIT, Layer

pytestmark = pytest.mark.gpu
F32, F16, BF16, F8, I8 = 0, 1, 30, 256, 24
KINDS, X_TYPES = M.KINDS, M.X_TYPES
NAMES = {F32: "f32", F16: "f16", BF16: "bf16", F8: "f8", I8: "i8"}
DISTINCT = 3


def matrix(kind, rng, groups, rows, k):
    """Experts of which every third is alike, with biases of their own."""
    if kind != I8:
        m = R.Matrix(kind, rng, groups, rows, k, True, distinct=DISTINCT)
        values = m.values
    else:
        m = Q.Matrix(rng, groups, rows, k, True, distinct=DISTINCT)
        m.scale_values = (m.scale_values * 15 / np.sqrt(k)).astype(np.float32)
        m.scales.upload(m.scale_values[np.arange(groups) % DISTINCT])
        values = m.codes * m.scale_values.astype(np.float64)[:, :, None]
    m.values = [values[g % DISTINCT] for g in range(groups)]
    return m


class WideLayer(Layer):
    def __init__(self, kind, E, H, I, K, act, seed):
        self.rng = np.random.default_rng(seed)
        self.E, self.H, self.I, self.K, self.act = E, H, I, K, act
        self.gu, self.dn = matrix(kind, self.rng, E, 2 * I, H), matrix(kind, self.rng, E, H, I)
        self.desc = vb.MoeFewDesc(self.gu.desc, self.dn.desc, K, act, ALPHA, LIMIT)


CASES = list(M.cases())


@pytest.mark.parametrize("kind,x_type,tokens,H,I", CASES, ids=[f"{NAMES[c[0]]}-{NAMES[c[1]]}-" + "_".join(map(str, (c[2], *M.kernel(*c[:3], c[4])))) for c in CASES])
def test_every_gate_up_kernel(gpu, kind, x_type, tokens, H, I):
    """Against float64, with the bounds of Layer.want and, since outputs are fp32, the norm of all errors."""
    L = WideLayer(kind, M.E, H, I, M.K, 1, seed=tokens + I)
    L.check(tokens, x_type, logits=(L.rng.standard_normal((tokens, M.E)) * 1.5).astype(np.float32))


def device_matrix(kind, values):
    """Weights [groups][rows][k] of -1, 0 and 1 as they are stored, their scales all 1."""
    groups, rows, k = values.shape
    scales = None
    if kind == F8:
        raw, scales = np.where(values == 0, 0, np.where(values < 0, 0xB8, 0x38)).astype(np.uint8), np.ones((groups, -(-rows // 128), -(-k // 128)), np.float32)
    elif kind == I8:
        raw, scales = values.astype(np.int8), np.ones((groups, rows), np.float32)
    else:
        raw = R.store_as(kind, values)[0]
    keep = [vb.DeviceBuffer.from_array(raw), vb.DeviceBuffer.from_array(scales) if scales is not None else None]
    return vb.Weights(kind, keep[0].ptr, vb.ptr(keep[1]), None, groups, rows, k), keep


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("x_type", X_TYPES)
@pytest.mark.parametrize("tokens", [1, 6])
def test_every_term_of_tokens_and_hidden_values_counts(gpu, kind, x_type, tokens):
    """Sums and differences that are exact in fp32 and cancel all but the last term of a value. Gates of 64 (whose sigmoid is 1 in fp32: e^-64 is below
    half a step of 1) make h = 64 up; 1 + 2^-9 + 2^-20 has bits in each of a value's three terms, 1 + 2^-7 + 2^-10 in both of an fp16 value's."""
    H, I = 272, 144
    full, less = {F32: (1 + 2.0 ** -9 + 2.0 ** -20, 1 + 2.0 ** -9), F16: (1 + 2.0 ** -7 + 2.0 ** -10, 1 + 2.0 ** -7), BF16: (1 + 2.0 ** -7, 1.0)}[x_type]
    x = np.zeros((tokens, H))
    x[:, [0, 5, 130, 131, 271]] = [full, 64.0, less, 1.0, 2.0 ** -9]
    x[:, 200] = 2.0 ** -20
    x *= np.where(np.arange(tokens) % 2, -1.0, 1.0)[:, None]
    x[:, 5] = 64.0
    gate, up, down = np.zeros((I, H)), np.zeros((I, H)), np.zeros((H, I))
    gate[:, 5] = 1
    up[0, 0], up[0, 130] = 1, -1                          # the token's last term alone
    up[7, 0] = 1
    up[100, [131, 271, 200]], up[143, [131, 271]] = 1, 1  # 1 + 2^-9 + 2^-20 and 1 + 2^-9, of any type of tokens
    down[0, 0], down[15, 7] = 1, 1
    down[16, 100], down[16, 143] = 1, -1                  # h's last term alone
    down[17, [100, 143]] = 1
    down[271, 100] = -1
    d1, keep1 = device_matrix(kind, np.concatenate([gate, up])[None])
    d2, keep2 = device_matrix(kind, down[None])
    L = Layer.__new__(Layer)
    L.H, L.I, L.K, L.E, L.desc = H, I, 1, 1, vb.MoeFewDesc(d1, d2, 1, 0, ALPHA, LIMIT)
    raw, v = R.store_as(x_type, x)
    assert np.array_equal(v, x)
    got, _, _ = L.run(tokens, x_type, raw, ids=np.zeros((tokens, 1), np.int32), weights=np.ones((tokens, 1), np.float32))
    want = 64 * (x @ up.T) @ down.T
    assert np.array_equal(want.astype(np.float32).astype(np.float64), want) and np.count_nonzero(want[0]) == 5
    assert np.array_equal(got, want), np.argwhere(got != want)[:4]


@pytest.mark.parametrize("kind", KINDS)
def test_wide_ranges_token_by_token(gpu, kind):
    """Tiny values next to large ones, and one token 2^40 times the others: each token's errors are held to its own norm, by 4e-6 as the whole of a layer's is."""
    H, I, T = 128, 64, 4
    L = Layer(kind, 4, H, I, 2, 0, False, seed=13)
    x = L.rng.standard_normal((T, H)).astype(np.float32) * np.exp2(L.rng.integers(-40, 8, (T, H))).astype(np.float32)
    x[1] *= np.float32(2.0 ** 40)
    ids, weights = np.array([[0, 1], [2, 3], [1, 1], [3, 0]], np.int32), np.full((T, 2), 0.5, np.float32)
    got, _, _ = L.run(T, F32, x, ids=ids, weights=weights)
    y, b = L.want(x.astype(np.float64), ids, weights, F32)
    err = np.abs(got - y)
    assert (err <= b).all()
    assert (np.linalg.norm(err, axis=1) <= 4e-6 * np.linalg.norm(y, axis=1)).all(), np.linalg.norm(err, axis=1) / np.linalg.norm(y, axis=1)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("x_type", X_TYPES)
@pytest.mark.parametrize("act", [0, 1])
def test_infinities(gpu, kind, x_type, act):
    """A token with an infinity of either sign comes out as NaN, as the formula has it here (some gates are -inf, and 0 times that is NaN); the
    others, of the same experts, as if it were not there."""
    L = Layer(kind, 2, 272, 80, 2, act, True, seed=14)
    T = 6
    x = L.rng.standard_normal((T, 272))
    x[1, 0], x[3, 271], x[4, 100] = np.inf, -np.inf, np.inf
    raw, v = R.store_as(x_type, x)
    ids, weights = np.tile(np.array([[0, 1]], np.int32), (T, 1)), np.full((T, 2), 0.5, np.float32)
    got, _, _ = L.run(T, x_type, raw, ids=ids, weights=weights)
    good, bad = [0, 2, 5], [1, 3, 4]
    y, b = L.want(v[good], ids[good], weights[good], F32)
    assert (np.abs(got[good] - y) <= b).all()
    with np.errstate(all="ignore"):
        assert np.isnan(L.want(v[bad], ids[bad], weights[bad], F32)[0]).all()
    assert np.isnan(got[bad]).all()


@pytest.mark.parametrize("kind,code,size", [(F8, 0x7E, 111), (I8, 127, 113)])
@pytest.mark.parametrize("x_type", [F32, BF16])
def test_sums_of_codes_up_to_the_end_of_fp32(gpu, kind, code, size, x_type):
    """The largest codes times tokens of 2^size, in sums of 128 just below 2^127, whose scale brings them back to 112 (e4m3's 448) or 127. Their sigmoid is 1 in
    fp32, and sums of the hidden values' squares are exact."""
    H, I, T = 128, 64, 3
    gu, dn = np.full((1, 2 * I, H), code, np.uint8), np.full((1, H, I), 0x38 if kind == F8 else 1, np.uint8)
    s1 = np.full((1, 1, 1) if kind == F8 else (1, 2 * I), 2.0 ** -120, np.float32)
    s2 = np.ones((1, 1, 1) if kind == F8 else (1, H), np.float32)
    d = [vb.DeviceBuffer.from_array(a) for a in (gu, s1, dn, s2)]
    L = Layer.__new__(Layer)
    L.H, L.I, L.K, L.E = H, I, 1, 1
    L.desc = vb.MoeFewDesc(vb.Weights(kind, d[0].ptr, d[1].ptr, None, 1, 2 * I, H), vb.Weights(kind, d[2].ptr, d[3].ptr, None, 1, H, I), 1, 0, ALPHA, LIMIT)
    raw, _ = R.store_as(x_type, np.full((T, H), 2.0 ** size))
    got, _, _ = L.run(T, x_type, raw, ids=np.zeros((T, 1), np.int32), weights=np.ones((T, 1), np.float32))
    gate = {F8: 448, I8: 127}[kind] * 128 * 2.0 ** (size - 120)
    assert gate in (112, 127) and (got == I * gate * gate).all()
