"""Arguments that the FP8 and grouped products refuse, before any device is touched; and the oracle of their tests
against itself."""
import numpy as np
import pytest

import fp8_ref as R

F32, F16, BF16, F8 = 0, 1, 30, 256
P = 4096                                        # an aligned address that nothing here dereferences


def status(vb, name, *args):
    return getattr(vb.load(), name)(*args)


def weights(vb, **kw):
    d = dict(type=F8, data=P, scales=P, bias=None, n_groups=1, rows=64, k=256)
    d.update(kw)
    return vb.Weights(*d.values())


@pytest.mark.parametrize("args,needle", [
    ((8, P, 4, 128, 128, P, P, None), b"F32, F16 or BF16"),
    ((F32, P, 4, 120, 128, P, P, None), b"multiple of 16"),
    ((F32, P, 4, 0, 128, P, P, None), b"multiple of 16"),
    ((F32, P, -1, 128, 128, P, P, None), b"multiple of 16"),
    ((F32, P, 4, 128, 112, P, P, None), b"k elements apart"),
    ((F32, None, 4, 128, 128, P, P, None), b"null"),
    ((F32, P, 4, 128, 128, None, P, None), b"null"),
    ((F32, P, 4, 128, 128, P, None, None), b"null"),
    ((F32, P + 2, 4, 128, 128, P, P, None), b"aligned"),
    ((BF16, P + 1, 4, 128, 128, P, P, None), b"aligned"),
    ((F32, P, 4, 128, 128, P + 8, P, None), b"aligned"),
    ((F32, P, 4, 128, 128, P, P + 2, None), b"aligned"),
    ((F32, P, 1 << 31, 128, 128, P, P, None), b"too many"),
])
def test_quantizer_refusals(vb, args, needle):
    assert status(vb, "vbm_quantize_fp8", *args) == 1
    assert needle in vb.load().vbm_last_error(), vb.load().vbm_last_error()


@pytest.mark.parametrize("args,needle", [
    ((2, F32, P, P, 4, 128, 128, 128, 1.0, 1.0, P, P, None), b"activation"),
    ((0, 39, P, P, 4, 128, 128, 128, 1.0, 1.0, P, P, None), b"F32, F16 or BF16"),
    ((0, F32, P, None, 4, 128, 128, 128, 1.0, 1.0, P, P, None), b"null"),
    ((0, F32, P, P, 4, 128, 128, 64, 1.0, 1.0, P, P, None), b"apart"),
    ((0, F32, P, P, 4, 72, 128, 128, 1.0, 1.0, P, P, None), b"multiple of 16"),
])
def test_glu_quantizer_refusals(vb, args, needle):
    assert status(vb, "vbm_glu_quantize_fp8", *args) == 1
    assert needle in vb.load().vbm_last_error(), vb.load().vbm_last_error()


@pytest.mark.parametrize("kw,call,needle", [
    (dict(type=39), {}, b"F8_E4M3"),
    (dict(type=BF16), {}, b"one F8_E4M3 matrix"),
    (dict(n_groups=2), {}, b"one F8_E4M3 matrix"),
    (dict(k=250), {}, b"multiple of 16"),
    (dict(k=0), {}, b"out of range"),
    (dict(rows=0), {}, b"out of range"),
    (dict(data=None), {}, b"null"),
    (dict(scales=None), {}, b"null"),
    (dict(data=P + 8), {}, b"16-byte"),
    (dict(bias=P + 2), {}, b"aligned"),
    ({}, dict(b=None), b"null"),
    ({}, dict(scales=None), b"null"),
    ({}, dict(b=P + 4), b"16-byte"),
    ({}, dict(tokens=-1), b"out of range"),
    ({}, dict(tokens=1 << 31), b"out of range"),
    ({}, dict(dst_type=8), b"dst must be"),
    ({}, dict(dst=None), b"null"),
    ({}, dict(dst=P + 2), b"aligned"),
])
def test_dense_refusals(vb, kw, call, needle):
    c = dict(b=P, scales=P, tokens=4, dst_type=F32, dst=P)
    c.update(call)
    assert status(vb, "vbm_mul_mat_fp8", weights(vb, **kw), *c.values(), None) == 1
    assert needle in vb.load().vbm_last_error(), vb.load().vbm_last_error()


@pytest.mark.parametrize("kw,call,needle", [
    (dict(type=F32), {}, b"F8_E4M3, F16 or BF16"),
    (dict(type=F16, k=100), {}, b"multiple of 8"),
    (dict(n_groups=0), {}, b"n_groups"),
    (dict(n_groups=1025), {}, b"n_groups"),
    ({}, dict(offsets=None), b"offsets"),
    ({}, dict(b_div=0), b"b_div"),
    ({}, dict(n_b=0), b"null"),
    ({}, dict(n_b=-1), b"out of range"),
    ({}, dict(n_rows=1 << 29), b"out of range"),
    ({}, dict(n_dst=-1), b"out of range"),
    ({}, dict(b_scales=None), b"null"),
    ({}, dict(b_rows=P + 2), b"aligned"),
    ({}, dict(dst_rows=P + 1), b"aligned"),
    ({}, dict(offsets=P + 1), b"aligned"),
])
def test_grouped_refusals(vb, kw, call, needle):
    c = dict(b=P, b_scales=P, n_b=8, b_rows=None, b_div=1, offsets=P, n_rows=8, dst_rows=None, n_dst=8, dst_type=F32, dst=P)
    c.update(call)
    assert status(vb, "vbm_grouped_mul_mat", weights(vb, **{"n_groups": 4, **kw}), *c.values(), None) == 1
    assert needle in vb.load().vbm_last_error(), vb.load().vbm_last_error()


def test_nothing_to_do_is_not_an_error(vb):
    assert status(vb, "vbm_quantize_fp8", F32, None, 0, 128, 128, None, None, None) == 0
    assert status(vb, "vbm_glu_quantize_fp8", 0, F32, None, None, 0, 128, 128, 128, 1.0, 1.0, None, None, None) == 0
    assert status(vb, "vbm_mul_mat_fp8", weights(vb), None, None, 0, F32, None, None) == 0
    assert status(vb, "vbm_grouped_mul_mat", weights(vb, n_groups=4), None, None, 0, None, 1, None, 0, None, 0, F32, None, None) == 0
    assert status(vb, "vbm_mul_mat_fp8", None, P, P, 4, F32, P, None) == 1
    assert status(vb, "vbm_grouped_mul_mat", None, P, P, 4, None, 1, P, 4, None, 4, F32, P, None) == 1


def test_reference_rounding_is_the_nearest_code():
    """e4m3_round against a search over all codes."""
    rng = np.random.default_rng(3)
    q = np.concatenate([rng.standard_normal(2000) * 100, np.exp2(rng.uniform(-12, 8.8, 2000)), R.E4M3[:127], (R.E4M3[:126] + R.E4M3[1:127]) / 2])
    q = np.clip(q, -448, 448)
    d = np.abs(q[:, None] - np.where(np.isnan(R.E4M3), np.inf, R.E4M3)[None, :])
    near = d == d.min(axis=1, keepdims=True)
    got = R.e4m3_round(q)
    assert near[np.arange(q.size), got].all()
    ties = near.sum(axis=1) > 1
    assert ((got[ties] & 1) == 0).all() or (R.E4M3[got[ties]] == 0).all()
