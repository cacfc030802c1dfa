"""Every kernel of the grouped product, for each kind of sums: values, root mean square errors, repeated calls, rows out of range, outputs
aligned to their type only, values that are not numbers."""
import numpy as np
import pytest

import fp8_ref as R
import product_cases as P
import vbmoe as vb

pytestmark = pytest.mark.gpu
F32, F16, BF16, F8 = 0, 1, 30, 256
CASES = list(P.cases())
IDS = [f"{t[0]}-{t[1]}-{name.replace(' ', '_')}" for t, name, *_ in CASES]
N_B = 301


class Call:
    """Random counts that add up to groups * mean rows, tokens taken from N_B distinct ones, outputs scattered; two rows are left over."""

    def __init__(self, types, groups, mean, rows, k, seed):
        rng = np.random.default_rng(seed)
        self.rng, self.dst_type = rng, types[1]
        self.n_rows = groups * mean
        self.counts = rng.multinomial(self.n_rows - 2, rng.dirichlet(np.full(groups, 4.0)))
        self.offsets = np.concatenate([[0], np.cumsum(self.counts)]).astype(np.int32)
        self.m, self.x = R.Matrix(types[0], rng, groups, rows, k, bias=True, distinct=min(3, groups)), R.Tokens(types[0], rng, N_B, k)
        self.b_rows = rng.integers(0, 2 * N_B, self.n_rows).astype(np.int32)
        self.dst_rows = rng.permutation(self.n_rows).astype(np.int32)

    @property
    def kw(self):
        return dict(b_rows=self.b_rows, b_div=2, dst_rows=self.dst_rows)

    def got(self):
        return R.grouped(self.m, self.x, N_B, self.offsets, self.n_rows, self.dst_type, self.n_rows, **self.kw)

    def want(self):
        return R.grouped_want(self.m, self.x, N_B, self.offsets, self.n_rows, self.n_rows, **self.kw)


def rms_bound(types, k, few):
    """Root mean square error over the outputs' own. fp32: k and some additions, each off by at most a step (2^-23) of a partial sum whose size grows
    with its root, in either direction: 2^-23 sqrt(k / 2). The FP8 instruction: seven of eight products lose less than 2^-13 of the largest, in
    either direction, a variance of 7/3 * 2^-26 of the largest's square, which is at most the eight's sum of squares, the
    variance of their sum: 1.9e-4. The output's rounding: at most half a step, evenly spread: over the root of 3."""
    err = (2.0 ** -23) ** 2 * (k + 128) / 2 + (R.HALF_STEP[types[1]] ** 2 / 3 if types[1] != F32 else 0.0)
    if P.KINDS[types] == 1 and not few:
        err += 7 / 3 * 2.0 ** -26
    return np.sqrt(err) * 1.02                          # (sums over some ten thousand outputs scatter by a percent)


@pytest.mark.parametrize("types,name,groups,mean,rows,k", CASES, ids=IDS)
def test_values_and_errors(gpu, types, name, groups, mean, rows, k):
    c = Call(types, groups, mean, rows, k, seed=len(name) * 100 + types[0] + types[1])
    got, (y, size, written) = c.got(), c.want()
    R.check(c.m, types[1], got, y, size, written, name)
    rms = np.sqrt(np.mean((got[written] - y[written]) ** 2) / np.mean(y[written] ** 2))
    bound = rms_bound(types, k, mean <= 10)
    print(f"[{name}] rms {rms:.3g} of {bound:.3g}", flush=True)
    assert rms <= bound


@pytest.mark.parametrize("types,name,groups,mean,rows,k", [c for c in CASES if c[0] in ((F8, F32), (F8, BF16), (F16, F16))],
                         ids=[i for i, c in zip(IDS, CASES) if c[0] in ((F8, F32), (F8, BF16), (F16, F16))])
def test_a_call_between_others_gives_the_same_bits(gpu, types, name, groups, mean, rows, k):
    """Three calls on one stream, another product and a quantizer before each but the first, their results read at the end."""
    c = Call(types, groups, mean, rows, k, seed=7)
    other = Call((F8, BF16), 4, 300, 1100, 400, seed=8)
    dev = lambda a: vb.DeviceBuffer.from_array(np.asarray(a, np.int32))  # noqa: E731
    size = c.n_rows * rows * R.SIZE[types[1]]
    outs, other_out = [R.filled(size) for _ in range(3)], R.filled(other.n_rows * 1100 * 2)
    bufs = {id(x): (dev(x.offsets), dev(x.b_rows), dev(x.dst_rows)) for x in (c, other)}
    noise = vb.DeviceBuffer.from_array(np.ones((512, 4096), np.float32))
    codes, scales = vb.DeviceBuffer(512 * 4096), vb.DeviceBuffer(512 * 32 * 4)

    def enqueue(x, out):
        off, b, d = bufs[id(x)]
        vb.call("vbm_grouped_mul_mat", x.m.desc, x.x.data.ptr, vb.ptr(x.x.scales), N_B, b.ptr, 2, off.ptr, x.n_rows, d.ptr, x.n_rows, x.dst_type, out.ptr, None)

    vb.call("vbm_stream_synchronize", None)
    for i, out in enumerate(outs):
        if i:
            enqueue(other, other_out)
            vb.call("vbm_quantize_fp8", F32, noise.ptr, 512, 4096, 4096, codes.ptr, scales.ptr, None)
        enqueue(c, out)
    vb.call("vbm_stream_synchronize", None)
    first, *rest = [out.download(np.uint8, (size,)) for out in outs]
    assert all(np.array_equal(first, r) for r in rest)


@pytest.mark.parametrize("types,name,groups,mean,rows,k", CASES, ids=IDS)
def test_rows_out_of_range_and_outputs_aligned_to_their_type(gpu, types, name, groups, mean, rows, k):
    """Source rows outside b give NaN, target rows outside dst are not written, offsets past n_rows end there; the outputs start
    one element into their buffer."""
    c = Call(types, groups, mean, rows, k, seed=9)
    c.offsets[-1] += 50                                 # (the last group then ends at n_rows)
    pick = c.rng.permutation(c.n_rows)
    c.b_rows[pick[:3]] = [-1, 2 * N_B, 2 ** 31 - 1]
    c.dst_rows[pick[3:5]] = [-1, c.n_rows]
    dev = lambda a: vb.DeviceBuffer.from_array(np.asarray(a, np.int32))  # noqa: E731
    off, b, d = dev(c.offsets), dev(c.b_rows), dev(c.dst_rows)
    es = R.SIZE[types[1]]
    size = c.n_rows * rows * es
    dst = R.filled(es + size + 32)
    vb.call("vbm_grouped_mul_mat", c.m.desc, c.x.data.ptr, vb.ptr(c.x.scales), N_B, b.ptr, 2, off.ptr, c.n_rows, d.ptr, c.n_rows, types[1], dst.ptr + es, None)
    vb.call("vbm_stream_synchronize", None)
    raw = dst.download(np.uint8, (dst.nbytes,))
    assert (raw[:es] == R.FILL).all() and (raw[es + size:] == R.FILL).all()
    out = raw[es:es + size].copy()
    got = {F32: lambda: out.view(np.float32), F16: lambda: out.view(np.float16), BF16: lambda: R.bf16_values(out.view(np.uint16))}[types[1]]()
    R.check(c.m, types[1], got.astype(np.float64).reshape(c.n_rows, rows), *c.want(), name)


@pytest.mark.parametrize("dst_type", [BF16, F16])
@pytest.mark.parametrize("tokens,rows", [(4, 160), (100, 160), (400, 160), (2000, 5200), (7, 65536 + 80)])
def test_values_that_are_not_numbers_in_16_bit_outputs(gpu, dst_type, tokens, rows):
    """NaN codes, NaN scales and infinite scales reach the outputs that read them, and no others."""
    rng = np.random.default_rng(5)
    k = 400
    codes, ws = R.fp8_matrix(rng, 1, rows, k)
    x, bs = R.quantize(rng.standard_normal((tokens, k)).astype(np.float32))
    codes[0, 7, 399] = 0x7F
    x[1, 0] = 0xFF
    bs[2, 1] = np.nan
    bs[3, 3] = np.inf
    d = [vb.DeviceBuffer.from_array(a) for a in (codes, ws, x, bs)]
    dst = vb.DeviceBuffer(tokens * rows * 2)
    vb.call("vbm_mul_mat_fp8", vb.Weights(F8, d[0].ptr, d[1].ptr, None, 1, rows, k), d[2].ptr, d[3].ptr, tokens, dst_type, dst.ptr, None)
    vb.call("vbm_stream_synchronize", None)
    want = np.ones((tokens, rows), bool)
    want[:, 7] = False
    want[1:4] = False
    assert np.array_equal(np.isfinite(R.load_as(dst_type, dst, (tokens, rows))), want)
