"""Arguments that the integer rows and products and the norm refuse, before any device is touched; the rule by which the integer products
choose their kernel; and the tests' own quantizer against float64."""
import subprocess
from fractions import Fraction
from pathlib import Path

import numpy as np
import pytest

import i8_ref as Q
import product_cases as P

REPO = Path(__file__).resolve().parents[1]
F32, F16, BF16, F8, I8 = 0, 1, 30, 256, 24
A = 4096                                        # an aligned address that nothing here dereferences


def refused(vb, needle, name, *args):
    assert getattr(vb.load(), name)(*args) == 1
    assert needle in vb.load().vbm_last_error(), vb.load().vbm_last_error()


@pytest.mark.parametrize("args,needle", [
    ((8, A, 4, 128, 128, A, A, None), b"F32, F16 or BF16"),
    ((F32, A, 4, 120, 128, A, A, None), b"multiple of 16"),
    ((F32, A, 4, 0, 128, A, A, None), b"multiple of 16"),
    ((F32, A, 4, 65536 + 16, 1 << 20, A, A, None), b"at most 65536"),
    ((F32, A, -1, 128, 128, A, A, None), b"n_rows"),
    ((F32, A, 1 << 31, 128, 128, A, A, None), b"n_rows"),
    ((F32, A, 4, 128, 112, A, A, None), b"k elements apart"),
    ((F32, A, 4, 128, 1 << 62, A, A, None), b"k elements apart"),
    ((F32, None, 4, 128, 128, A, A, None), b"null"),
    ((F32, A, 4, 128, 128, None, A, None), b"null"),
    ((F32, A, 4, 128, 128, A, None, None), b"null"),
    ((F32, A + 2, 4, 128, 128, A, A, None), b"aligned"),
    ((BF16, A + 1, 4, 128, 128, A, A, None), b"aligned"),
    ((F32, A, 4, 128, 128, A + 8, A, None), b"aligned"),
    ((F32, A, 4, 128, 128, A, A + 2, None), b"aligned"),
])
def test_quantizer_refusals(vb, args, needle):
    refused(vb, needle, "vbm_quantize_i8", *args)


@pytest.mark.parametrize("args,needle", [
    ((2, F32, A, A, 4, 128, 128, 128, 1.0, 1.0, A, A, None), b"activation"),
    ((0, 39, A, A, 4, 128, 128, 128, 1.0, 1.0, A, A, None), b"F32, F16 or BF16"),
    ((0, F32, A, None, 4, 128, 128, 128, 1.0, 1.0, A, A, None), b"null"),
    ((0, F32, A, A, 4, 128, 128, 64, 1.0, 1.0, A, A, None), b"apart"),
    ((0, F32, A, A, 4, 128, 64, 128, 1.0, 1.0, A, A, None), b"apart"),
    ((0, F32, A, A, 4, 72, 128, 128, 1.0, 1.0, A, A, None), b"multiple of 16"),
    ((0, BF16, A, A + 1, 4, 128, 128, 128, 1.0, 1.0, A, A, None), b"aligned"),
])
def test_glu_quantizer_refusals(vb, args, needle):
    refused(vb, needle, "vbm_glu_quantize_i8", *args)


NORM = dict(x_type=BF16, x=A, x_stride=128, residual=A, sum=A, residual_stride=128, weight=A, n_rows=4, k=128, eps=1e-6, y_type=BF16, y=A,
            code_type=I8, codes=A, scales=A, stream=None)


@pytest.mark.parametrize("change,needle", [
    (dict(x_type=39), b"x must be F32, F16 or BF16"), (dict(y_type=I8), b"y must be F32, F16 or BF16"), (dict(code_type=F16), b"F8_E4M3 or I8"),
    (dict(k=120), b"multiple of 16"), (dict(k=65552, x_stride=1 << 20, residual_stride=1 << 20), b"at most 65536"), (dict(n_rows=-1), b"n_rows"),
    (dict(x=None), b"null"), (dict(x_stride=64), b"apart"), (dict(residual_stride=64), b"apart"), (dict(residual=None), b"without a residual"),
    (dict(eps=0.0), b"eps"), (dict(eps=-1.0), b"eps"), (dict(eps=float("nan")), b"eps"), (dict(eps=float("inf")), b"eps"),
    (dict(y=None, codes=None), b"neither"), (dict(scales=None), b"null"), (dict(x=A + 1), b"aligned"), (dict(residual=A + 1), b"aligned"),
    (dict(sum=A + 1), b"aligned"), (dict(weight=A + 2), b"aligned"), (dict(y=A + 1), b"aligned"), (dict(codes=A + 8), b"aligned"),
    (dict(scales=A + 1), b"aligned"),
])
def test_norm_refusals(vb, change, needle):
    refused(vb, needle, "vbm_add_rms_norm_quantize", *{**NORM, **change}.values())


def weights(vb, **kw):
    return vb.Weights(*{**dict(type=I8, data=A, scales=A, bias=None, n_groups=1, rows=64, k=256), **kw}.values())


@pytest.mark.parametrize("kw,call,needle", [
    (dict(type=F8), {}, b"one I8 matrix"), (dict(type=BF16), {}, b"one I8 matrix"), (dict(n_groups=2), {}, b"one I8 matrix"),
    (dict(k=250), {}, b"multiple of 16"), (dict(k=131072), {}, b"less than 131072"), (dict(rows=0), {}, b"out of range"),
    (dict(data=None), {}, b"null"), (dict(scales=None), {}, b"null"), (dict(data=A + 8), {}, b"16-byte"), (dict(scales=A + 2), {}, b"aligned"),
    (dict(bias=A + 2), {}, b"aligned"), ({}, dict(b=None), b"null"), ({}, dict(scales=None), b"null"), ({}, dict(b=A + 4), b"16-byte"),
    ({}, dict(tokens=-1), b"out of range"), ({}, dict(tokens=1 << 29), b"out of range"), ({}, dict(dst_type=I8), b"dst must be"),
    ({}, dict(dst=None), b"null"), ({}, dict(dst=A + 2), b"aligned"),
])
def test_dense_refusals(vb, kw, call, needle):
    refused(vb, needle, "vbm_mul_mat_i8", weights(vb, **kw), *{**dict(b=A, scales=A, tokens=4, dst_type=F32, dst=A), **call}.values(), None)


@pytest.mark.parametrize("kw,call,needle", [
    (dict(scales=None), {}, b"null"), (dict(k=131072), {}, b"less than 131072"), (dict(k=24), {}, b"multiple of 16"),
    ({}, dict(b_scales=None), b"null"), ({}, dict(offsets=None), b"offsets"), ({}, dict(n_rows=1 << 29), b"out of range"),
])
def test_grouped_refusals(vb, kw, call, needle):
    c = dict(b=A, b_scales=A, n_b=8, b_rows=None, b_div=1, offsets=A, n_rows=8, dst_rows=None, n_dst=8, dst_type=F32, dst=A)
    refused(vb, needle, "vbm_grouped_mul_mat", weights(vb, **{"n_groups": 4, **kw}), *{**c, **call}.values(), None)


def test_nothing_to_do_is_not_an_error(vb):
    lib = vb.load()
    assert lib.vbm_quantize_i8(F32, None, 0, 128, 128, None, None, None) == 0
    assert lib.vbm_glu_quantize_i8(0, F32, None, None, 0, 128, 128, 128, 1.0, 1.0, None, None, None) == 0
    assert lib.vbm_mul_mat_i8(weights(vb), None, None, 0, F32, None, None) == 0
    assert lib.vbm_mul_mat_i8(None, A, A, 4, F32, A, None) == 1
    none = dict(x=None, residual=None, sum=None, y=None, codes=None, scales=None, weight=None, n_rows=0)
    assert lib.vbm_add_rms_norm_quantize(*{**NORM, **none}.values()) == 0


# ---------------------------------------------------------------------------------- kernel choice
def cases():
    """Calls that reach every kernel of the grouped product: its groups, rows a group, weight rows and k for codes of a byte."""
    for name, (groups, mean, rows, k) in {**P.FEW, **P.DEEP, **P.MANY}.items():
        yield name, groups, mean, rows, DEPTHS.get(name, k[8] if isinstance(k, dict) else k)


# (the integers' scales leave room for deeper tokens than the FP8 blocks' do)
DEPTHS = {"stream8_8": 6032, "stream16_8": 4624, "few16 past LDS": 6032, "few8 past LDS": 12048}


def test_every_case_reaches_the_kernel_it_is_for(tmp_path):
    exe = tmp_path / "rule"
    subprocess.run(["g++", "-O2", "-std=c++17", f"-I{REPO / 'unified-memory-scheduler_amd' / 'csrc'}",
                    str(REPO / "tests" / "cpp" / "test_i8_product_rule.cpp"), "-o", str(exe)], check=True)
    calls = [(1, g * mean, g, rows, k) for _, g, mean, rows, k in cases()]
    out = subprocess.run([str(exe)], input="".join(" ".join(map(str, c)) + "\n" for c in calls), capture_output=True, text=True, check=True, timeout=60)
    assert out.stdout.split() == [name.split()[0] for name, *_ in cases()]


# ------------------------------------------------------------------------------------ the oracle
def test_reference_codes_are_the_rounded_quotients():
    """The fp32 steps against whole fractions: 127 x / a rounded once to fp32 (16-bit inputs make 127 x exact) and then to an integer."""
    rng = np.random.default_rng(5)
    x = np.concatenate([rng.standard_normal((20, 48)), rng.integers(-127, 128, (20, 48)) / 2, np.zeros((1, 48))]).astype(np.float16).astype(np.float32)
    codes, scales = Q.quantize(x)
    for row, c, s in zip(x, codes, scales):
        a = max(np.float32(np.abs(row).max()), np.float32(2.0 ** -116))
        assert s == np.float32(float(a) / 127)
        for v, got in zip(row, c):
            q = Fraction(float(v)) * 127 / Fraction(float(a))
            near = np.float32(float(q))                     # (float64 first: a double rounding here would need 29 equal bits)
            assert got == int(np.rint(near)) and abs(Fraction(int(got)) - q) <= Fraction(1, 2) + abs(q) / 2 ** 23
