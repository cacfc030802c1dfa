"""The FP8 quantizers and the dense and grouped products on the GPU against float64 forms (fp8_ref)."""
import ctypes as C

import numpy as np
import pytest

import fp8_ref as R
import vbmoe as vb

pytestmark = pytest.mark.gpu
F32, F16, BF16, F8 = 0, 1, 30, 256
TYPES = [F32, F16, BF16]


def sync(stream=None):
    vb.call("vbm_stream_synchronize", stream)


# ------------------------------------------------------------------------------------- quantizers
def quantize(type_id, x, k, stride=None, offset=0):
    """codes, scales of rows that start `offset` elements into their buffer, `stride` apart; checks that nothing
    behind them is written."""
    rows = x.shape[0]
    stride = stride or k
    raw, _ = R.store_as(type_id, x)
    host = np.zeros(offset + rows * stride, raw.dtype)
    host[offset:].reshape(rows, stride)[:, :k] = raw
    dx = vb.DeviceBuffer.from_array(host)
    kb = -(-k // 128)
    dc, ds = R.filled(rows * k + 64), R.filled(4 * rows * kb + 64)
    vb.call("vbm_quantize_fp8", type_id, dx.ptr + offset * R.SIZE[type_id], rows, k, stride, dc.ptr, ds.ptr, None)
    sync()
    codes, scales = dc.download(np.uint8, (dc.nbytes,)), ds.download(np.uint8, (ds.nbytes,))
    assert (codes[rows * k:] == R.FILL).all() and (scales[4 * rows * kb:] == R.FILL).all()
    return codes[:rows * k].reshape(rows, k), scales[:4 * rows * kb].view(np.float32).reshape(rows, kb)


def same_codes(codes, scales, want_c, want_s):
    assert np.array_equal(scales.view(np.uint32), want_s.view(np.uint32)) or np.array_equal(np.nan_to_num(scales, nan=-1), np.nan_to_num(want_s, nan=-1))
    bad = np.argwhere(codes != want_c)
    assert not len(bad), (len(bad), bad[:4], codes[tuple(bad[0])], want_c[tuple(bad[0])])


@pytest.mark.parametrize("type_id", TYPES)
@pytest.mark.parametrize("rows,k,stride,offset", [(1, 16, None, 0), (1, 2880, None, 0), (3, 128, None, 0), (37, 592, None, 0),
                                                  (300, 768, 1536, 0), (5, 144, 147, 3), (2, 8192, None, 8), (17, 48, 50, 1)])
def test_quantize_equals_the_definition(gpu, type_id, rows, k, stride, offset):
    rng = np.random.default_rng(rows * 1000 + k)
    x = rng.standard_normal((rows, k)).astype(np.float32) * np.exp2(rng.integers(-12, 12, (rows, 1))).astype(np.float32)
    _, v = R.store_as(type_id, x)
    same_codes(*quantize(type_id, x, k, stride, offset), *R.quantize(v))


@pytest.mark.parametrize("type_id", TYPES)
def test_quantize_special_values(gpu, type_id):
    """Zeros, ties, subnormals, the largest values, and blocks with NaN or infinities beside ordinary ones."""
    k = 400
    rng = np.random.default_rng(11)
    x = rng.standard_normal((12, k)).astype(np.float32)
    big = {F32: 3.4e38, F16: 65504.0, BF16: 3.3e38}[type_id]
    x[0] = 0.0
    x[1, :128] = -0.0
    x[2] = np.round(x[2] * 8) / 8                                        # ties of the e4m3 grid
    x[2, ::128] = 7.0
    x[3, 5], x[3, 200] = np.nan, np.inf
    x[4, 399] = -np.inf                                                  # in the short last block
    x[5] *= np.float32(1e-30)
    x[6] *= np.float32(1e-37)
    x[7] = big * np.sign(x[7])
    x[8, 0] = big
    x[9, 127], x[9, 128] = 448.0, -448.0
    x[10, :] = np.float32(2.0) ** rng.integers(-20, 10, k)
    x[11, 1:] = 0.0
    _, v = R.store_as(type_id, x)
    codes, scales = quantize(type_id, x, k)
    same_codes(codes, scales, *R.quantize(v))
    assert np.isnan(scales[3, :2]).all() and np.isnan(scales[4, 3]) and np.isfinite(scales[4, :3]).all()


def glu_values(act, g, u, alpha, limit):
    if act == 1:
        g, u = np.minimum(g, limit), np.clip(u, -limit, limit)
        with np.errstate(over="ignore"):
            return g / (1 + np.exp(-alpha * g)) * (u + 1)
    with np.errstate(over="ignore"):
        return g / (1 + np.exp(-g)) * u


@pytest.mark.parametrize("type_id", TYPES)
@pytest.mark.parametrize("act", [0, 1])
@pytest.mark.parametrize("rows,width,extra,offset,size", [(1, 16, 0, 0, 1), (8, 768, 0, 0, 3), (33, 2880, 0, 0, 10), (5, 208, 5, 1, 60)])
def test_glu_quantize(gpu, type_id, act, rows, width, extra, offset, size):
    """Within half a step of e4m3 of the float64 value, and the scale within the fp32 arithmetic's error: the argument of the exponential
    is rounded (2^-24 of it, which is a relative error of |argument| 2^-24 in the result), and eight more roundings follow."""
    rng = np.random.default_rng(width + act)
    alpha, limit, stride = 1.702, 7.0, 2 * width + extra
    x = rng.standard_normal((rows, stride)).astype(np.float32) * size
    x[0, :8] = 0.0
    if size >= 10:
        x[0, 8], x[0, 9] = -200.0, -95.0                                 # exponentials past the fp32 range
    raw, v = R.store_as(type_id, x)
    host = np.zeros(offset + raw.size, raw.dtype)
    host[offset:] = raw.reshape(-1)
    dx = vb.DeviceBuffer.from_array(host)
    kb, es = -(-width // 128), R.SIZE[type_id]
    dc, ds = R.filled(rows * width + 64), R.filled(4 * rows * kb + 64)
    vb.call("vbm_glu_quantize_fp8", act, type_id, dx.ptr + offset * es, dx.ptr + (offset + width) * es, rows, width, stride, stride,
            alpha, limit, dc.ptr, ds.ptr, None)
    sync()
    assert (dc.download(np.uint8, (dc.nbytes,))[rows * width:] == R.FILL).all()
    codes, scales = dc.download(np.uint8, (rows, width)), ds.download(np.float32, (rows, kb)).astype(np.float64)
    h = glu_values(act, v[:, :width], v[:, width:2 * width], float(np.float32(alpha)), limit)
    a = np.maximum(np.abs(R.blocks_of(h)).max(axis=2), float(R.LEAST))
    rel = (np.abs(v[:, :width]).max() * alpha + 8) * 2.0 ** -24
    assert (np.abs(scales - a / 448) <= rel * a / 448).all()
    q = R.blocks_of(h) * (448 / a)[:, :, None]
    size_q = np.maximum(np.abs(q), 2.0 ** -6)
    half = np.exp2(np.floor(np.log2(size_q))) / 16
    got = R.blocks_of(R.E4M3[codes])
    assert (np.abs(got - q) <= half * (1 + 1e-4) + 2 * rel * 448).all()


def test_glu_quantize_marks_blocks_without_a_scale(gpu):
    width = 256
    x = np.ones((3, 2 * width), np.float32)
    x[1, 3] = np.nan                                                     # gate
    x[2, width + 200] = np.inf                                           # up: SiLU keeps it
    dx, dc, ds = vb.DeviceBuffer.from_array(x), vb.DeviceBuffer(3 * width), vb.DeviceBuffer(24)
    vb.call("vbm_glu_quantize_fp8", 0, F32, dx.ptr, dx.ptr + 4 * width, 3, width, 2 * width, 2 * width, 1.702, 7.0, dc.ptr, ds.ptr, None)
    sync()
    scales, codes = ds.download(np.float32, (3, 2)), dc.download(np.uint8, (3, width))
    assert np.array_equal(np.isnan(scales), [[False, False], [True, False], [False, True]])
    assert (codes[1, :128] == 0).all() and (codes[2, 128:] == 0).all() and (codes[0] == 0x7E).all()


# ---------------------------------------------------------------------------------- dense product
@pytest.mark.parametrize("dst_type", TYPES)
@pytest.mark.parametrize("tokens,rows,k,bias", [(1, 64, 128, False), (1, 300, 2880, True), (2, 1, 16, True), (15, 129, 48, False), (16, 15, 144, False),
                                                (17, 100, 336, True), (40, 130, 2048, False), (65, 257, 720, True), (130, 515, 400, False),
                                                (300, 384, 1040, True), (2085, 6164, 144, True), (1000, 2000, 272, False),
                                                (3, 70, 8720, True), (9, 33, 8832, False), (300, 130, 8720, True), (2500, 4100, 8336, False)])
def test_dense_product(gpu, dst_type, tokens, rows, k, bias):
    rng = np.random.default_rng(tokens * 31 + rows)
    m, x = R.Matrix(F8, rng, 1, rows, k, bias), R.Tokens(F8, rng, tokens, k)
    dst = R.filled((tokens + 1) * rows * R.SIZE[dst_type])
    vb.call("vbm_mul_mat_fp8", m.desc, x.data.ptr, x.scales.ptr, tokens, dst_type, dst.ptr, None)
    sync()
    got = R.load_as(dst_type, dst, (tokens + 1, rows))
    y, size, written = R.grouped_want(m, x, tokens, [0, tokens], tokens, tokens + 1)
    R.check(m, dst_type, got, y, size, written, f"dense {tokens}x{rows}x{k}")


# -------------------------------------------------------------------------------- grouped product
SIZES = {
    "one row": [0, 1, 0],
    "empty ends": [0, 0, 5, 0, 17, 0],
    "tile edges": [16, 15, 33, 1, 64, 63, 65],
    "one takes all": [0, 0, 150, 0],
    "large": [300, 0, 129, 257, 31],
    "no rows": [0, 0, 0],
}


@pytest.mark.parametrize("type_id", [F8, F16, BF16])
@pytest.mark.parametrize("dst_type", [F32, BF16])
@pytest.mark.parametrize("sizes", list(SIZES))
@pytest.mark.parametrize("gather", [True, False])
def test_grouped_product(gpu, type_id, dst_type, sizes, gather):
    """Gathered tokens (each row's token is rows / top_k) into grouped order, and grouped rows scattered to their (token, rank) places;
    the last rows belong to no group and stay as they were."""
    counts = SIZES[sizes]
    rng = np.random.default_rng(len(sizes) * 7 + type_id + gather)
    used = sum(counts)
    n_rows = used + 3
    rows, k, top_k = 200, 336, 4
    m = R.Matrix(type_id, rng, len(counts), rows, k, bias=gather)
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    place = rng.permutation(n_rows).astype(np.int32)
    n_b = -(-n_rows // top_k) if gather else n_rows
    x = R.Tokens(type_id, rng, n_b, k)
    kw = dict(b_rows=place, b_div=top_k) if gather else dict(dst_rows=place)
    got = R.grouped(m, x, n_b, offsets, n_rows, dst_type, n_rows, **kw)
    R.check(m, dst_type, got, *R.grouped_want(m, x, n_b, offsets, n_rows, n_rows, **kw), f"grouped {sizes}")


@pytest.mark.parametrize("type_id", [F8, BF16])
@pytest.mark.parametrize("groups", [1, 63, 64, 65, 200, 1024])
def test_grouped_product_over_many_groups(gpu, type_id, groups):
    rng = np.random.default_rng(groups)
    counts = rng.integers(0, 3, groups)
    counts[rng.integers(0, groups)] = 40
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    used = int(offsets[-1])
    m, x = R.Matrix(type_id, rng, groups, 33, 128), R.Tokens(type_id, rng, used, 128)
    got = R.grouped(m, x, used, offsets, used, F32, used)
    R.check(m, F32, got, *R.grouped_want(m, x, used, offsets, used, used), f"{groups} groups")


@pytest.mark.parametrize("type_id,dst_type", [(F8, F32), (F8, BF16), (F16, F16), (BF16, F32)])
@pytest.mark.parametrize("groups,rows,k,most", [(140, 481, 336, 16), (1024, 64, 1808, 3), (70, 1037, 3296, 19), (300, 250, 6800, 9), (500, 161, 1024, 33)])
def test_grouped_product_few_rows_of_many(gpu, type_id, dst_type, groups, rows, k, most):
    """Some rows for each of many experts, at depths whose tokens do and do not fit on the chip."""
    k = k if type_id == F8 else k // 2
    rng = np.random.default_rng(groups + k)
    counts = rng.integers(0, most + 1, groups)
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    n_rows = int(offsets[-1]) + 2
    place = rng.permutation(n_rows).astype(np.int32)
    gather = k % 32 == 0
    n_b = -(-n_rows // 2) if gather else n_rows
    m, x = R.Matrix(type_id, rng, groups, rows, k, bias=True, distinct=4), R.Tokens(type_id, rng, n_b, k)
    kw = dict(b_rows=place, b_div=2) if gather else dict(dst_rows=place)
    got = R.grouped(m, x, n_b, offsets, n_rows, dst_type, n_rows, **kw)
    R.check(m, dst_type, got, *R.grouped_want(m, x, n_b, offsets, n_rows, n_rows, **kw), f"few rows of {groups}")


@pytest.mark.parametrize("type_id,dst_type", [(F8, F32), (F8, F16), (F8, BF16), (F16, F32), (BF16, BF16)])
@pytest.mark.parametrize("gather", [True, False])
@pytest.mark.parametrize("rows,k,groups,most", [(2100, 272, 24, 290), (1090, 400, 24, 290), (520, 656, 6, 290), (257, 1168, 3, 700)])
def test_grouped_product_many_rows(gpu, type_id, dst_type, gather, rows, k, groups, most):
    """Sizes from a few rows to several tiles a group, in launches that fill the card and small ones."""
    rng = np.random.default_rng(rows + k + gather)
    counts = np.concatenate([[0, 1, 2 * most // 3], rng.integers(0, most, groups)])[:groups]
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    n_rows, top_k = int(offsets[-1]) + 5, 3
    place = rng.permutation(n_rows).astype(np.int32)
    n_b = -(-n_rows // top_k) if gather else n_rows
    m, x = R.Matrix(type_id, rng, groups, rows, k, bias=not gather), R.Tokens(type_id, rng, n_b, k)
    kw = dict(b_rows=place, b_div=top_k) if gather else dict(dst_rows=place)
    got = R.grouped(m, x, n_b, offsets, n_rows, dst_type, n_rows, **kw)
    R.check(m, dst_type, got, *R.grouped_want(m, x, n_b, offsets, n_rows, n_rows, **kw), f"many rows {rows}x{k}")


@pytest.mark.parametrize("dst_type,offset", [(F32, 4), (F32, 8), (F16, 2), (BF16, 6), (BF16, 8)])
@pytest.mark.parametrize("tokens,rows", [(2, 64), (30, 72), (333, 256)])
def test_outputs_that_are_aligned_to_their_type_only(gpu, dst_type, offset, tokens, rows):
    rng = np.random.default_rng(offset + tokens)
    k = 208
    m, x = R.Matrix(F8, rng, 1, rows, k, True), R.Tokens(F8, rng, tokens, k)
    size = R.SIZE[dst_type]
    dst = R.filled(16 + tokens * rows * size + 64)
    vb.call("vbm_mul_mat_fp8", m.desc, x.data.ptr, x.scales.ptr, tokens, dst_type, dst.ptr + offset, None)
    sync()
    raw = dst.download(np.uint8, (dst.nbytes,))
    end = offset + tokens * rows * size
    assert (raw[:offset] == R.FILL).all() and (raw[end:] == R.FILL).all()
    out = raw[offset:end].copy()
    got = {F32: lambda: out.view(np.float32), F16: lambda: out.view(np.float16), BF16: lambda: R.bf16_values(out.view(np.uint16))}[dst_type]()
    y, mag, written = R.grouped_want(m, x, tokens, [0, tokens], tokens, tokens)
    R.check(m, dst_type, got.astype(np.float64).reshape(tokens, rows), y, mag, written, "unaligned outputs")


def test_a_call_gives_the_same_bits_again(gpu):
    """Few, some and many rows a group: repeated calls, with other work between them, give equal bits."""
    rng = np.random.default_rng(21)
    for type_id, counts, rows, k in ((F8, [3, 1, 2], 100, 528), (F8, [60, 0, 33], 640, 1040), (BF16, [300, 200], 1100, 264), (F8, [9] * 70, 1000, 400)):
        offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        n = int(offsets[-1])
        m, x = R.Matrix(type_id, rng, len(counts), rows, k), R.Tokens(type_id, rng, n, k)
        first = R.grouped(m, x, n, offsets, n, F32, n)
        for _ in range(3):
            assert np.array_equal(R.grouped(m, x, n, offsets, n, F32, n), first)


@pytest.mark.parametrize("type_id", [F8, F16])
@pytest.mark.parametrize("count", [9, 150, 700])
def test_rows_out_of_range(gpu, type_id, count):
    """A source row outside b gives NaN outputs, a target row outside dst is not written, and offsets past n_rows end there."""
    rng = np.random.default_rng(count)
    n_b, n_dst, rows, k = 50, count + 4, 72, 272
    m, x = R.Matrix(type_id, rng, 2, rows, k), R.Tokens(type_id, rng, n_b, k)
    b_rows = rng.integers(0, n_b, count).astype(np.int32)
    dst_rows = rng.permutation(n_dst)[:count].astype(np.int32)
    b_rows[[0, 4, count - 1]] = [-1, n_b, 2**31 - 1]
    dst_rows[[2, 5]] = [-1, n_dst]
    offsets = np.array([0, count // 3, count + 100], np.int32)
    kw = dict(b_rows=b_rows, dst_rows=dst_rows)
    got = R.grouped(m, x, n_b, offsets, count, F32, n_dst, **kw)
    R.check(m, F32, got, *R.grouped_want(m, x, n_b, offsets, count, n_dst, **kw), "out of range")


@pytest.mark.parametrize("tokens", [4, 100, 400])
def test_values_that_are_not_numbers(gpu, tokens):
    """NaN codes, NaN scales and infinite scales reach the outputs that read them, and no others."""
    rng = np.random.default_rng(5)
    rows, k = 160, 400
    codes, ws = R.fp8_matrix(rng, 1, rows, k)
    x, bs = R.quantize(rng.standard_normal((tokens, k)).astype(np.float32))
    codes[0, 7, 399] = 0x7F
    x[1, 0] = 0xFF
    bs[2, 1] = np.nan
    bs[3, 3] = np.inf
    d = [vb.DeviceBuffer.from_array(a) for a in (codes, ws, x, bs)]
    dst = vb.DeviceBuffer(tokens * rows * 4)
    vb.call("vbm_mul_mat_fp8", vb.Weights(F8, d[0].ptr, d[1].ptr, None, 1, rows, k), d[2].ptr, d[3].ptr, tokens, F32, dst.ptr, None)
    sync()
    got = dst.download(np.float32, (tokens, rows))
    want = np.ones((tokens, rows), bool)
    want[:, 7] = False
    want[1:4] = False
    assert np.array_equal(np.isfinite(got), want)


# --------------------------------------------------------------------------- together, in a layer
def fp8_layer(dev, rng, T, H, I, E, K, act):
    """The routed FFN of one layer with FP8 experts, as the calls are meant to be chained. Returns a function that enqueues it
    and the buffers."""
    gu, dn = R.Matrix(F8, rng, E, 2 * I, H, True), R.Matrix(F8, rng, E, H, I, True)
    x = rng.standard_normal((T, H)).astype(np.float32)
    logits = rng.standard_normal((T, E)).astype(np.float32)
    n = T * K
    b = {name: vb.DeviceBuffer(size) for name, size in dict(
        ids=4 * n, weights=4 * n, counts=4 * E, offsets=4 * (E + 1), rows=4 * n, xc=T * H, xs=4 * T * -(-H // 128), gu=2 * n * 2 * I,
        hc=n * I, hs=4 * n * -(-I // 128), y=4 * n * H, out=4 * T * H).items()}
    b["x"], b["logits"] = vb.DeviceBuffer.from_array(x), vb.DeviceBuffer.from_array(logits)

    def enqueue(s):
        p = {name: buf.ptr for name, buf in b.items()}
        vb.call("vbm_router_topk_softmax", None, None, None, 0, p["logits"], E, T, K, p["ids"], p["weights"], s)
        vb.call("vbm_group_by_expert", p["ids"], K, T, K, E, p["counts"], p["offsets"], p["rows"], None, s)
        vb.call("vbm_quantize_fp8", F32, p["x"], T, H, H, p["xc"], p["xs"], s)
        vb.call("vbm_grouped_mul_mat", gu.desc, p["xc"], p["xs"], T, p["rows"], K, p["offsets"], n, None, n, BF16, p["gu"], s)
        vb.call("vbm_glu_quantize_fp8", act, BF16, p["gu"], p["gu"] + 2 * I, n, I, 2 * I, 2 * I, 1.702, 7.0, p["hc"], p["hs"], s)
        vb.call("vbm_grouped_mul_mat", dn.desc, p["hc"], p["hs"], n, None, 1, p["offsets"], n, p["rows"], n, F32, p["y"], s)
        vb.call("vbm_weighted_combine", p["y"], p["weights"], H, K, T, p["out"], s)
    return enqueue, b, gu, dn, x, logits


@pytest.mark.parametrize("T,H,I,E,K,act", [(1, 256, 192, 8, 2, 0), (5, 2880, 336, 8, 4, 1), (200, 512, 400, 8, 4, 1)])
def test_layer_of_fp8_experts(gpu, T, H, I, E, K, act):
    """The chain against float64 on the same quantized input. Between the two products the activations are rounded to e4m3, off by at most
    half a step, 2^-4 of the value (2^-10 of a code's unit for the smallest); the gate and up values before that to bf16. An output
    is held to what those roundings can add up to through |down|, and (far closer) the whole to their root mean square."""
    rng = np.random.default_rng(T + H)
    stream = C.c_void_p()
    vb.call("vbm_stream_create", C.byref(stream))
    enqueue, b, gu, dn, x, logits = fp8_layer(gpu, rng, T, H, I, E, K, act)
    enqueue(stream.value)
    sync(stream.value)
    got = b["out"].download(np.float32, (T, H)).astype(np.float64)
    xq = R.rows_of(*R.quantize(x))
    order = np.argsort(-logits, axis=1, kind="stable")[:, :K]
    want, bound = np.zeros((T, H)), np.zeros((T, H))
    for t in range(T):
        z = logits[t, order[t]].astype(np.float64)
        w = np.exp(z - z.max()) / np.exp(z - z.max()).sum()
        for j, e in enumerate(order[t]):
            g = gu.values[e] @ xq[t] + gu.bias_values[e]
            h = glu_values(act, g[:I], g[I:], 1.702, 7.0)
            want[t] += w[j] * (dn.values[e] @ h + dn.bias_values[e])
            # bf16 gate and up (2^-8 each; |d glu / d gate| <= 1.13 (|up| + 1), |d glu / d up| <= |gate|), then e4m3
            a = np.abs(R.blocks_of(h[None])).max(axis=2).repeat(128, axis=1)[0, :I]
            dh = 2.0 ** -8 * (1.2 * np.abs(g[:I]) * (np.abs(g[I:]) + 1) + np.abs(g[:I]) * np.abs(g[I:])) * 1.01
            dh = dh + 2.0 ** -4 * 1.01 * (np.abs(h) + dh) + a / 448 * 2.0 ** -10 + 2.0 ** -8 * a * 2.0 ** -4
            bound[t] += w[j] * (np.abs(dn.values[e]) @ dh + 1e-4)
    err = np.abs(got - want)
    assert (err <= bound).all(), float((err / bound).max())
    rel = np.linalg.norm(got - want) / np.linalg.norm(want)
    print(f"[fp8 layer T={T}] rel {rel:.4f}", flush=True)
    assert rel <= 2.0 ** -4
    vb.call("vbm_stream_destroy", stream.value)


def test_captured_layer_replays_on_new_inputs(gpu):
    """One graph of the chain, replayed with new tokens between eager calls on another stream: the eager results' bits."""
    rng = np.random.default_rng(77)
    T, H, I, E, K = 40, 512, 256, 8, 2
    s1, s2, graph = C.c_void_p(), C.c_void_p(), C.c_void_p()
    vb.call("vbm_stream_create", C.byref(s1))
    vb.call("vbm_stream_create", C.byref(s2))
    enqueue, b, gu, dn, x, logits = fp8_layer(gpu, rng, T, H, I, E, K, 1)
    enqueue(s1.value)                                   # (the grouping's scratch is allocated by a first call)
    sync(s1.value)
    vb.call("vbm_graph_begin_capture", s1.value)
    enqueue(s1.value)
    vb.call("vbm_graph_end_capture", s1.value, C.byref(graph))
    for step in range(4):
        b["x"].upload(rng.standard_normal((T, H)).astype(np.float32), s1.value)
        b["logits"].upload(rng.standard_normal((T, E)).astype(np.float32), s1.value)
        enqueue(s2.value)
        sync(s2.value)
        want = b["out"].download(np.uint32, (T, H))
        vb.call("vbm_memset", b["out"].ptr, 0, b["out"].nbytes, s1.value)
        sync(s1.value)
        vb.call("vbm_graph_launch", graph.value, s1.value)
        sync(s1.value)
        assert np.array_equal(b["out"].download(np.uint32, (T, H)), want), step
    vb.call("vbm_graph_destroy", graph.value)
    vb.call("vbm_stream_destroy", s1.value)
    vb.call("vbm_stream_destroy", s2.value)


def test_two_streams_at_once(gpu):
    """The same calls in flight on two streams give what they give alone."""
    rng = np.random.default_rng(78)
    streams, layers = [C.c_void_p(), C.c_void_p()], []
    for s in streams:
        vb.call("vbm_stream_create", C.byref(s))
        layers.append(fp8_layer(gpu, rng, 64, 512, 256, 8, 2, 0))
    alone = []
    for s, (enqueue, b, *_) in zip(streams, layers):
        enqueue(s.value)
        sync(s.value)
        alone.append(b["out"].download(np.uint32, (64, 512)))
    for _ in range(3):
        for _ in range(4):
            for s, (enqueue, *_) in zip(streams, layers):
                enqueue(s.value)
        for s in streams:
            sync(s.value)
        for want, (_, b, *_) in zip(alone, layers):
            assert np.array_equal(b["out"].download(np.uint32, (64, 512)), want)
    for s in streams:
        vb.call("vbm_stream_destroy", s.value)
