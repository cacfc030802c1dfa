"""Arguments that the layer for a few tokens refuses, before any device is touched, and the size of its workspace."""
import ctypes as C

import pytest

F32, F16, BF16, F8, I8 = 0, 1, 30, 256, 24
A = 4096                                        # an aligned address that nothing here dereferences


def desc(vb, gate_up=None, down=None, **kw):
    g = {**dict(type=F8, data=A, scales=A, bias=None, n_groups=8, rows=512, k=128), **(gate_up or {})}
    d = {**dict(type=F8, data=A, scales=A, bias=None, n_groups=8, rows=128, k=256), **(down or {})}
    return vb.MoeFewDesc(vb.Weights(*g.values()), vb.Weights(*d.values()), *{**dict(top_k=2, activation=0, alpha=1.702, limit=7.0), **kw}.values())


@pytest.mark.parametrize("kw,tokens,needle", [
    (dict(gate_up=dict(type=F32)), 1, b"I8, F8_E4M3, F16 or BF16"), (dict(down=dict(type=I8)), 1, b"one type"),
    (dict(gate_up=dict(n_groups=0)), 1, b"experts"), (dict(gate_up=dict(n_groups=1025), down=dict(n_groups=1025)), 1, b"experts"),
    (dict(down=dict(n_groups=7)), 1, b"experts"), (dict(gate_up=dict(rows=500)), 1, b"[2 * I][H]"), (dict(down=dict(rows=112)), 1, b"[2 * I][H]"),
    (dict(gate_up=dict(k=120), down=dict(rows=120)), 1, b"multiples of 16"), (dict(gate_up=dict(rows=496), down=dict(k=248)), 1, b"multiples of 16"),
    (dict(gate_up=dict(type=BF16, k=124), down=dict(type=BF16, rows=124)), 1, b"multiples of 8"),
    (dict(gate_up=dict(k=0), down=dict(rows=0)), 1, b"out of range"), (dict(gate_up=dict(rows=1 << 24), down=dict(k=1 << 23)), 1, b"out of range"),
    (dict(gate_up=dict(data=None)), 1, b"null"), (dict(down=dict(scales=None)), 1, b"null"), (dict(gate_up=dict(data=A + 8)), 1, b"16-byte"),
    (dict(down=dict(scales=A + 2)), 1, b"aligned"), (dict(gate_up=dict(bias=A + 1)), 1, b"aligned"),
    (dict(activation=2), 1, b"activation"), (dict(top_k=0), 1, b"top_k"), (dict(top_k=9), 1, b"top_k"),
    ({}, -1, b"16 tokens"), ({}, 17, b"16 tokens"), (dict(gate_up=dict(n_groups=64), down=dict(n_groups=64), top_k=9), 15, b"128 (token, rank) pairs"),
    (dict(gate_up=dict(n_groups=128), down=dict(n_groups=128), top_k=65), 1, b"top_k"),
])
def test_description_refusals(vb, kw, tokens, needle):
    size = C.c_size_t()
    assert vb.load().vbm_moe_few_workspace(desc(vb, **kw), tokens, size) == 1
    assert needle in vb.load().vbm_last_error(), vb.load().vbm_last_error()
    assert vb.load().vbm_moe_few_forward(desc(vb, **kw), F32, A, A, A, A, tokens, F32, A, A, 1 << 30, None) == 1
    assert needle in vb.load().vbm_last_error(), vb.load().vbm_last_error()


CALL = dict(x_type=BF16, x=A, logits=A, ids=A, weights=A, tokens=4, out_type=BF16, out=A, workspace=A, size=1 << 20, stream=None)


@pytest.mark.parametrize("change,needle", [
    (dict(x_type=I8), b"x must be"), (dict(out_type=F8), b"out must be"), (dict(x=None), b"null"), (dict(out=None), b"null"), (dict(workspace=None), b"null"),
    (dict(logits=None, ids=None), b"neither"), (dict(logits=None, weights=None), b"neither"), (dict(x=A + 8), b"16-byte"), (dict(workspace=A + 8), b"16-byte"),
    (dict(out=A + 1), b"aligned"), (dict(logits=A + 2), b"aligned"), (dict(ids=A + 2), b"aligned"), (dict(weights=A + 2), b"aligned"),
    (dict(size=1024 + 8 * 2 * 768 - 1), b"too small"),
])
def test_call_refusals(vb, change, needle):
    assert vb.load().vbm_moe_few_forward(desc(vb), *{**CALL, **change}.values()) == 1
    assert needle in vb.load().vbm_last_error(), vb.load().vbm_last_error()


def test_nothing_to_do_is_not_an_error(vb):
    none = dict(x=None, logits=None, ids=None, weights=None, tokens=0, out=None, workspace=None, size=0)
    assert vb.load().vbm_moe_few_forward(desc(vb), *{**CALL, **none}.values()) == 0
    assert vb.load().vbm_moe_few_forward(None, *CALL.values()) == 1
    assert vb.load().vbm_moe_few_workspace(desc(vb), 1, None) == 1


@pytest.mark.parametrize("kind,tokens,top_k,inter,want", [
    (F8, 1, 2, 256, 1024 + 2 * 2 * 768), (I8, 4, 2, 272, 1024 + 8 * 3 * 768), (BF16, 16, 8, 72, 1024 + 128 * 2 * 384), (F16, 0, 2, 64, 1024),
])
def test_workspace(vb, kind, tokens, top_k, inter, want):
    """Six bytes a value of h, whole steps of 128 or 64 values, behind the routing's kilobyte."""
    size = C.c_size_t()
    vb.call("vbm_moe_few_workspace", desc(vb, dict(type=kind, rows=2 * inter), dict(type=kind, k=inter), top_k=top_k), tokens, size)
    assert size.value == want
