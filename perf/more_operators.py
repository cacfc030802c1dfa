"""Norms with quantized outputs, the 8-bit integer products and a whole layer of experts for a few tokens, as cases that
can be timed and checked one by one.

A case is a dict of plain values; `op` names the operator:

- "norm": a block's output added to the residual stream, the root-mean-square norm of the sum, and that as 8-bit codes
  with scales (vbm_add_rms_norm_quantize): e4m3 with one scale per 128 values, or integers with one per row;
- "rows": rows of activations, or an expert's gated activation (`glu`), to 8-bit integers with one scale per row
  (vbm_quantize_i8, vbm_glu_quantize_i8);
- "dense": the product of 8-bit integer weights, one scale per output channel, with such rows (vbm_mul_mat_i8);
- "grouped": the same for tokens grouped by expert, ragged (vbm_grouped_mul_mat with integer weights). `gather`: the gate_up
  side, which reads each token's row for every expert it is routed to and writes in grouped order; else the down side, which
  reads grouped order and writes each (token, rank) row to its place;
- "layer": all of a routed-expert layer for a few tokens, from router logits (or a given routing) to the weighted sum of the
  experts' outputs, the weights as they are stored (vbm_moe_few_forward).

Where `own` is false, `run` computes the same in elementary torch operations, in 32 bits.

8-bit integer codes that depend on a sum or an exponential come back times their scales, as bf16 values (torch has no type
for them); the codes of plain rows, which are defined to the bit, as they are.
"""
import ctypes
import math
import sys
from pathlib import Path

import torch

own = False
DEVICE = "cuda"
TORCH_TYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPE_ID = {"f32": 0, "f16": 1, "i8": 24, "bf16": 30, "f8": 256}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "f8": 1, "i8": 1}
SILU, OAI = 0, 1
ALPHA, LIMIT = 1.702, 7.0
EPS = 1e-6
BLOCK = 128
MOST = {"f8": 448.0, "i8": 127.0}   # the largest code's value
LEAST = 2.0 ** -116                 # values that are all smaller share this one's scale


def listed():
    return [
        # one token between two layers of a decode step, before FP8 experts: latency
        {"name": "norm_1x2880_f8", "op": "norm", "rows": 1, "k": 2880, "type": "bf16", "codes": "f8"},
        # an odd-sized prompt before integer products
        {"name": "norm_1517x2880_i8", "op": "norm", "rows": 1517, "k": 2880, "type": "f16", "codes": "i8"},
        # a large prefill batch
        {"name": "norm_8192x4096_f8", "op": "norm", "rows": 8192, "k": 4096, "type": "bf16", "codes": "f8"},
        # a prompt's attention outputs before an integer projection
        {"name": "rows_8192x4096_bf16", "op": "rows", "rows": 8192, "k": 4096, "type": "bf16", "glu": False, "act": SILU},
        # a decode batch between the two expert products: fused gate | up rows
        {"name": "glu_256x2880_f32", "op": "rows", "rows": 256, "k": 2880, "type": "f32", "glu": True, "act": OAI},
        # a dense projection of one decoded token: the weights are read once
        {"name": "dense_1x5760x2880", "op": "dense", "tokens": 1, "rows": 5760, "k": 2880, "bias": True, "out": "f32"},
        # a large prefill batch
        {"name": "dense_4096x4096x4096", "op": "dense", "tokens": 4096, "rows": 4096, "k": 4096, "bias": False, "out": "bf16"},
        # a decode batch: some rows for each of 32 experts, with biases
        {"name": "grouped_64", "op": "grouped", "tokens": 64, "top_k": 4, "experts": 32, "rows": 5760, "k": 2880,
         "gather": True, "bias": True, "masked": False, "out": "f32"},
        # prefill of an odd-sized prompt over 128 experts, the down side, some routes masked
        {"name": "grouped_1517", "op": "grouped", "tokens": 1517, "top_k": 8, "experts": 128, "rows": 2048, "k": 768,
         "gather": False, "bias": False, "masked": True, "out": "bf16"},
        # one decoded token through eight of 128 FP8 experts, from the router's logits
        {"name": "layer_f8_1", "op": "layer", "type": "f8", "tokens": 1, "top_k": 8, "experts": 128, "hidden": 2048, "inter": 768,
         "act": SILU, "bias": False, "routed": True, "x": "bf16"},
        # the same decode step over integer experts with biases, four tokens
        {"name": "layer_i8_4", "op": "layer", "type": "i8", "tokens": 4, "top_k": 4, "experts": 32, "hidden": 2880, "inter": 2880,
         "act": OAI, "bias": True, "routed": True, "x": "f32"},
        # a decode batch of sixteen tokens over 16-bit experts, the routing given
        {"name": "layer_bf16_16", "op": "layer", "type": "bf16", "tokens": 16, "top_k": 4, "experts": 32, "hidden": 2880, "inter": 2880,
         "act": OAI, "bias": True, "routed": False, "x": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "rows", "dense", "dense", "grouped", "grouped", "layer", "layer", "layer"])
    kind = rng.choice(["f32", "bf16", "f16"])
    if op in ("norm", "rows"):
        k, rows = 16 * _log_int(rng, 4, 512), _log_int(rng, 1, 16384)
        rows = max(1, min(rows, 8192 * 2048 // k))
        if op == "norm":
            return {"op": op, "rows": rows, "k": k, "type": kind, "codes": rng.choice(["f8", "i8"])}
        return {"op": op, "rows": rows, "k": k, "type": kind, "glu": rng.random() < 0.5, "act": rng.choice([SILU, OAI])}
    if op == "layer":
        experts, tokens = _log_int(rng, 4, 128), _log_int(rng, 1, 16)
        c = {"op": op, "type": rng.choice(["f8", "i8", "bf16", "f16"]), "tokens": tokens, "top_k": rng.randint(1, min(8, experts)),
             "experts": experts, "hidden": 16 * _log_int(rng, 8, 256), "inter": 16 * _log_int(rng, 8, 256), "act": rng.choice([SILU, OAI]),
             "bias": rng.random() < 0.5, "routed": rng.random() < 0.5, "x": kind}
        # no more weights than the listed ones hold and read
        while c["experts"] > c["top_k"] and 3.0 * c["experts"] * c["hidden"] * c["inter"] > 7.0e8:
            c["experts"] = max(c["top_k"], c["experts"] * 2 // 3)
        while c["tokens"] > 1 and 3.0 * min(c["experts"], c["tokens"] * c["top_k"]) * c["hidden"] * c["inter"] > 6.5e8:
            c["tokens"] = c["tokens"] * 2 // 3
        return c
    # row counts that are no multiple of anything now and then; depths are multiples of 16 values
    rows = rng.choice([_log_int(rng, 64, 6144), 64 * _log_int(rng, 1, 90)])
    k = 16 * _log_int(rng, 8, 400)
    c = {"op": op, "tokens": _log_int(rng, 1, 4096), "rows": rows, "k": k, "bias": rng.random() < 0.5, "out": kind}
    if op == "grouped":
        experts = _log_int(rng, 4, 128)
        c = {**c, "top_k": rng.randint(1, min(8, experts)), "experts": experts, "gather": rng.random() < 0.5, "masked": rng.random() < 0.5}
        while c["experts"] > c["top_k"] and 1.0 * c["experts"] * rows * k > 4.0e8:
            c["experts"] = max(c["top_k"], c["experts"] * 2 // 3)
    while c["tokens"] > 1 and 2.0 * c["tokens"] * c.get("top_k", 1) * rows * k > 1.0e11:
        c["tokens"] = c["tokens"] * 2 // 3
    return c


# ------------------------------------------------------------------------------------------ inputs
def _gen(seed, place):
    g = torch.Generator(device=DEVICE)
    g.manual_seed((seed * 1000003 + place * 7919 + 29) & 0x7FFFFFFFFFFF)
    return g


def _normal(seed, place, *shape, std=1.0):
    return torch.randn(*shape, generator=_gen(seed, place), device=DEVICE, dtype=torch.float32) * std


def _activations(seed, place, rows, k):
    """N(0, 1) with a few channels that are ten times as large, as hidden states have them."""
    channel = 1.0 + 9.0 * (torch.rand(k, generator=_gen(seed, place + 1), device=DEVICE) < 0.01)
    return _normal(seed, place, rows, k) * channel


def _weights(seed, place, kind, experts, rows, k):
    """(codes or values [experts][rows][k], scales or None) of normal weights: e4m3 with a scale per 128 x 128 block,
    integers with one per row, or 16-bit values."""
    if kind == "f8":
        nb, kb = -(-rows // BLOCK), -(-k // BLOCK)
        w = torch.zeros(experts, nb * BLOCK, kb * BLOCK, device=DEVICE)
        w[:, :rows, :k] = _normal(seed, place, experts, rows, k, std=1.0 / math.sqrt(k))
        blocks = w.view(experts, nb, BLOCK, kb, BLOCK)
        scales = blocks.abs().amax(dim=(2, 4)).clamp_(min=LEAST) / MOST["f8"]
        blocks /= scales[:, :, None, :, None]
        return w[:, :rows, :k].to(torch.float8_e4m3fn).view(torch.uint8).contiguous(), scales
    w = _normal(seed, place, experts, rows, k, std=1.0 / math.sqrt(k))
    if kind == "i8":
        scales = w.abs().amax(dim=2).clamp_(min=LEAST) / MOST["i8"]
        return w.div_(scales[:, :, None]).round_().to(torch.int8), scales
    return w.to(TORCH_TYPE[kind]), None


def _quantize_rows(x):
    """(int8 codes, scales) of fp32 rows."""
    most = x.abs().amax(dim=1, keepdim=True).clamp_(min=LEAST)
    return (x * MOST["i8"] / most).round().to(torch.int8), (most / MOST["i8"]).squeeze(1)


def _quantize_blocks(x):
    """(e4m3 codes, scales [rows][ceil(k / 128)]) of fp32 rows."""
    rows, k = x.shape
    kb = -(-k // BLOCK)
    v = torch.nn.functional.pad(x, (0, kb * BLOCK - k)).view(rows, kb, BLOCK)
    most = v.abs().amax(dim=2).clamp_(min=LEAST)
    codes = (v * MOST["f8"] / most[:, :, None]).to(torch.float8_e4m3fn)
    return codes.view(rows, kb * BLOCK)[:, :k].contiguous(), most / MOST["f8"]


class _State:
    pass


def prepare(case, seed):
    c, s = case, _State()
    s.case = c
    op = c["op"]
    if op in ("norm", "rows"):
        rows, k, t = c["rows"], c["k"], TORCH_TYPE[c["type"]]
        # (the fused product's rows: gate in the first half of each, up in the second)
        s.x = _activations(seed, 1, rows, 2 * k if c.get("glu") else k).to(t)
        if op == "norm":
            s.residual = (3.0 * _activations(seed, 3, rows, k)).to(t)
            s.weight = 0.5 + torch.rand(k, generator=_gen(seed, 5), device=DEVICE)
            s.sum, s.y = torch.empty_like(s.x), torch.empty_like(s.x)
        f8 = c.get("codes") == "f8"
        s.codes = torch.empty(rows, k, device=DEVICE, dtype=torch.float8_e4m3fn if f8 else torch.int8)
        s.scales = torch.empty((rows, -(-k // BLOCK)) if f8 else rows, device=DEVICE)
        s.values = None if f8 else torch.empty(rows, k, device=DEVICE, dtype=torch.bfloat16)
        return s
    if op == "layer":
        T, K, E, H, I, kind = c["tokens"], c["top_k"], c["experts"], c["hidden"], c["inter"], c["type"]
        s.w1, s.s1 = _weights(seed, 10, kind, E, 2 * I, H)
        s.w2, s.s2 = _weights(seed, 12, kind, E, H, I)
        s.b1 = _normal(seed, 20, E, 2 * I, std=0.1) if c["bias"] else None
        s.b2 = _normal(seed, 21, E, H, std=0.1) if c["bias"] else None
        s.x = _activations(seed, 1, T, H).to(TORCH_TYPE[c["x"]])
        s.logits = _normal(seed, 30, T, E, std=1.5)
        s.ids, s.weights = (v.contiguous() for v in _routing(s.logits, K))
        s.ids = s.ids.to(torch.int32)
        s.out = torch.empty_like(s.x)
        s.plan = None
        return s
    E, N, k = c.get("experts", 1), c["rows"], c["k"]
    s.w, s.ws = _weights(seed, 10, "i8", E, N, k)
    s.bias = _normal(seed, 20, E, N, std=0.02) if c["bias"] else None
    entries = c["tokens"] * c.get("top_k", 1)
    s.b, s.bs = _quantize_rows(_activations(seed, 1, c["tokens"] if op == "dense" or c["gather"] else entries, k))
    s.out = torch.zeros(entries, N, device=DEVICE, dtype=TORCH_TYPE[c["out"]])
    if op == "grouped":
        # experts are liked unequally; a masked route has none
        T, K = c["tokens"], c["top_k"]
        score = torch.rand(T, E, generator=_gen(seed, 30), device=DEVICE) + 0.05 * torch.rand(E, generator=_gen(seed, 31), device=DEVICE)
        ids = score.topk(K, dim=1).indices.reshape(-1)
        if c["masked"]:
            ids = torch.where(torch.rand(T * K, generator=_gen(seed, 32), device=DEVICE) < 0.03, torch.full_like(ids, E), ids)
        s.rows = torch.sort(ids, stable=True).indices.to(torch.int32)
        counts = torch.bincount(ids, minlength=E + 1)[:E]
        s.offsets = torch.zeros(E + 1, device=DEVICE, dtype=torch.int32)
        s.offsets[1:] = counts.cumsum(0)
        s.used, s.most, s.active = int(counts.sum()), int(counts.max()), counts.nonzero().squeeze(1)
    return s


# --------------------------------------------------------------------------------- the plain forms
def _routing(logits, top_k):
    """ids and weights of the top_k experts of each token, the softmax over those."""
    most = logits.topk(top_k, dim=1)
    e = torch.exp(most.values - most.values[:, :1])
    return most.indices, e / e.sum(dim=1, keepdim=True)


def _gated(act, g, u):
    if act == OAI:
        g, u = g.clamp(max=LIMIT), u.clamp(-LIMIT, LIMIT)
        return g / (1 + torch.exp(-ALPHA * g)) * (u + 1)
    return g / (1 + torch.exp(-g)) * u


def _values(w, ws):
    """fp32 weights [experts][rows][k] of stored ones and their scales."""
    if w.dtype == torch.int8:
        return w.float() * ws[:, :, None]
    if ws is None:
        return w.float()
    E, N, k = w.shape
    v = w.view(torch.float8_e4m3fn).float()
    by_k = ws.repeat_interleave(BLOCK, dim=2)[:, :, :k]
    whole = N // BLOCK * BLOCK
    if whole:
        v[:, :whole].unflatten(1, (-1, BLOCK)).mul_(by_k[:, :whole // BLOCK, None, :])
    if whole < N:
        v[:, whole:].mul_(by_k[:, -1:, :])
    return v


def _times(codes, scales):
    return (codes * scales[:, None]).to(torch.bfloat16)


def _plain(s):
    c = s.case
    if c["op"] == "norm":
        total = (s.x.float() + s.residual.float()).to(s.x.dtype)
        v = total.float()
        y = v * torch.rsqrt(v.square().mean(dim=1, keepdim=True) + EPS) * s.weight
        codes, scales = _quantize_blocks(y) if c["codes"] == "f8" else _quantize_rows(y)
        return {"sum": total, "y": y.to(s.x.dtype), "codes": codes if c["codes"] == "f8" else _times(codes, scales), "scales": scales}
    if c["op"] == "rows":
        x = s.x.float()
        codes, scales = _quantize_rows(_gated(c["act"], x[:, :c["k"]], x[:, c["k"]:]) if c["glu"] else x)
        return {"codes": _times(codes, scales) if c["glu"] else codes, "scales": scales}
    if c["op"] == "dense":
        y = (s.b.float() @ s.w[0].float().T) * (s.bs[:, None] * s.ws)
        if s.bias is not None:
            y += s.bias
        return {"out": y.to(TORCH_TYPE[c["out"]])}
    if c["op"] == "layer":
        T, K, I = c["tokens"], c["top_k"], c["inter"]
        ids, weights = _routing(s.logits, K) if c["routed"] else (s.ids.long(), s.weights)
        # one product for each (token, rank)
        e = ids.reshape(-1)
        at = lambda v: None if v is None else v[e]  # noqa: E731
        x = s.x.float().repeat_interleave(K, dim=0)
        g = torch.bmm(_values(s.w1[e], at(s.s1)), x[:, :, None]).squeeze(2)
        if s.b1 is not None:
            g += s.b1[e]
        h = _gated(c["act"], g[:, :I], g[:, I:])
        y = torch.bmm(_values(s.w2[e], at(s.s2)), h[:, :, None]).squeeze(2)
        if s.b2 is not None:
            y += s.b2[e]
        out = (y.view(T, K, -1) * weights[:, :, None]).sum(dim=1).to(s.x.dtype)
        return {"out": out, "ids": ids.to(torch.int32), "weights": weights} if c["routed"] else {"out": out}
    # the touched experts' rows side by side, padded to the longest, and one batched product
    k = c["k"]
    counts = s.offsets.diff()
    at = torch.arange(s.used, device=DEVICE, dtype=torch.int32)
    expert = torch.searchsorted(s.offsets[1:], at, right=True)
    slot, place = ((counts > 0).cumsum(0) - 1)[expert], at - s.offsets[expert]
    rows = s.rows[:s.used]
    src = rows // c["top_k"] if c["gather"] else at
    x = torch.zeros(len(s.active), s.most, k, device=DEVICE)
    x[slot, place] = s.b[src].float()
    y = torch.bmm(s.w[s.active].float(), x.transpose(1, 2).contiguous())[slot, :, place] * (s.bs[src][:, None] * s.ws[expert])
    if s.bias is not None:
        y += s.bias[expert]
    s.out[at if c["gather"] else rows] = y.to(s.out.dtype)
    return {"out": s.out}


# ---------------------------------------------------------------------------- this engine's kernels
def _engine():
    path = str(Path(__file__).resolve().parent.parent / "unified-memory-scheduler_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import vbmoe
    return vbmoe


def _ptr(t):
    return None if t is None else t.data_ptr()


def _kernels(s):
    vb, c = _engine(), s.case
    stream = torch.cuda.current_stream().cuda_stream
    op = c["op"]
    if op == "norm":
        kind, k = TYPE_ID[c["type"]], c["k"]
        vb.call("vbm_add_rms_norm_quantize", kind, s.x.data_ptr(), k, s.residual.data_ptr(), s.sum.data_ptr(), k, s.weight.data_ptr(),
                c["rows"], k, EPS, kind, s.y.data_ptr(), TYPE_ID[c["codes"]], s.codes.data_ptr(), s.scales.data_ptr(), stream)
        codes = s.codes if s.values is None else torch.mul(s.codes, s.scales[:, None], out=s.values)
        return {"sum": s.sum, "y": s.y, "codes": codes, "scales": s.scales}
    if op == "rows":
        kind, k, x = TYPE_ID[c["type"]], c["k"], s.x.data_ptr()
        if not c["glu"]:
            vb.call("vbm_quantize_i8", kind, x, c["rows"], k, k, s.codes.data_ptr(), s.scales.data_ptr(), stream)
            return {"codes": s.codes, "scales": s.scales}
        vb.call("vbm_glu_quantize_i8", c["act"], kind, x, x + k * BYTES[c["type"]], c["rows"], k, 2 * k, 2 * k, ALPHA, LIMIT,
                s.codes.data_ptr(), s.scales.data_ptr(), stream)
        return {"codes": torch.mul(s.codes, s.scales[:, None], out=s.values), "scales": s.scales}
    if op == "layer":
        E, H, I, kind = c["experts"], c["hidden"], c["inter"], TYPE_ID[c["type"]]
        if s.plan is None:
            s.plan = vb.MoeFewDesc(vb.Weights(kind, _ptr(s.w1), _ptr(s.s1), _ptr(s.b1), E, 2 * I, H),
                                   vb.Weights(kind, _ptr(s.w2), _ptr(s.s2), _ptr(s.b2), E, H, I), c["top_k"], c["act"], ALPHA, LIMIT)
            size = ctypes.c_size_t()
            vb.call("vbm_moe_few_workspace", s.plan, c["tokens"], size)
            s.workspace = torch.empty(size.value, device=DEVICE, dtype=torch.uint8)
        x = TYPE_ID[c["x"]]
        vb.call("vbm_moe_few_forward", s.plan, x, s.x.data_ptr(), s.logits.data_ptr() if c["routed"] else None, s.ids.data_ptr(),
                s.weights.data_ptr(), c["tokens"], x, s.out.data_ptr(), s.workspace.data_ptr(), s.workspace.numel(), stream)
        return {"out": s.out, "ids": s.ids, "weights": s.weights} if c["routed"] else {"out": s.out}
    w = vb.Weights(TYPE_ID["i8"], s.w.data_ptr(), s.ws.data_ptr(), _ptr(s.bias), s.w.shape[0], c["rows"], c["k"])
    out = TYPE_ID[c["out"]]
    if op == "dense":
        vb.call("vbm_mul_mat_i8", w, s.b.data_ptr(), s.bs.data_ptr(), c["tokens"], out, s.out.data_ptr(), stream)
    else:
        rows, gather, n = s.rows.data_ptr(), c["gather"], s.out.shape[0]
        vb.call("vbm_grouped_mul_mat", w, s.b.data_ptr(), s.bs.data_ptr(), s.b.shape[0], rows if gather else None,
                c["top_k"] if gather else 1, s.offsets.data_ptr(), n, None if gather else rows, n, out, s.out.data_ptr(), stream)
    return {"out": s.out}


def run(s):
    return _kernels(s) if own else _plain(s)


def work(case):
    c = case
    if c["op"] in ("norm", "rows"):
        rows, k = c["rows"], c["k"]
        scales = 4.0 * (-(-k // BLOCK) if c.get("codes") == "f8" else 1)
        if c["op"] == "norm":   # both inputs, the sum, the norm and its codes
            return {"bytes": rows * (k * (4.0 * BYTES[c["type"]] + 1) + scales) + 4.0 * k, "flops": rows * k * 8.0}
        halves = 2 if c["glu"] else 1
        return {"bytes": rows * (k * (halves * BYTES[c["type"]] + 1) + scales), "flops": rows * k * (12.0 if c["glu"] else 3.0)}
    if c["op"] == "layer":
        T, K, E, H, I, b = c["tokens"], c["top_k"], c["experts"], c["hidden"], c["inter"], BYTES[c["type"]]
        touched = E * (1 - (1 - K / E) ** T)
        scales = {"f8": 4.0 * (-(-2 * I // BLOCK) * -(-H // BLOCK) + -(-H // BLOCK) * -(-I // BLOCK)), "i8": 4.0 * (2 * I + H)}.get(c["type"], 0.0)
        return {"bytes": touched * (3.0 * H * I * b + scales + (4.0 * (2 * I + H) if c["bias"] else 0)) + 2.0 * T * H * BYTES[c["x"]]
                + (4.0 * T * E if c["routed"] else 8.0 * T * K), "flops": 6.0 * T * K * H * I}
    N, E, k = c["rows"], c.get("experts", 1), c["k"]
    entries = c["tokens"] * c.get("top_k", 1) * (0.97 if c.get("masked") else 1.0)
    touched = E * (1 - (1 - c["top_k"] / E) ** c["tokens"]) if c["op"] == "grouped" else 1
    n_b = c["tokens"] if c["op"] == "dense" or c["gather"] else entries
    lists = 4.0 * (entries + E + 1) if c["op"] == "grouped" else 0.0
    return {"bytes": touched * N * (k + 4.0 + (4.0 if c["bias"] else 0)) + n_b * (k + 4.0) + lists + entries * N * BYTES[c["out"]],
            "flops": 2.0 * entries * N * k}


# ---------------------------------------------------------------------------------- 64-bit values
def _e4m3_values(codes):
    """float64 values of e4m3 bytes, from the format: 4 exponent bits with bias 7, 3 mantissa bits."""
    v = codes.to(torch.int64)
    e, m = (v >> 3) & 15, (v & 7).double()
    size = torch.where(e > 0, (1 + m / 8) * torch.exp2(e.double() - 7), m / 8 * 2.0 ** -6)
    return torch.where(v >= 128, -size, size)


def _nearest_e4m3(x):
    """float64 values rounded to e4m3's grid, ties to even."""
    size = x.abs().clamp(min=1e-300)
    step = torch.exp2(torch.floor(torch.log2(size)).clamp(min=-6.0) - 3)
    return torch.round(x / step) * step


def _expand(scales, dim, size):
    return scales.double().index_select(dim, torch.arange(size, device=DEVICE) // BLOCK)


def _exact_matrix(w, ws, e):
    """float64 weights of expert e."""
    if ws is None:
        return w[e].double()
    if w.dtype == torch.int8:
        return w[e].double() * ws[e].double().unsqueeze(1)
    return _e4m3_values(w[e]) * _expand(_expand(ws[e], 0, w.shape[1]), 1, w.shape[2])


def _exact_glu(act, g, u):
    if act == OAI:
        g, u = torch.clamp(g, max=LIMIT), torch.clamp(u, -LIMIT, LIMIT)
        return g * torch.sigmoid(ALPHA * g) * (1 + u)
    return g * torch.sigmoid(g) * u


def _exact_codes(v, kind):
    """(values of the codes, not yet times the scales, and the scales)."""
    rows, k = v.shape
    if kind == "i8":
        most = torch.clamp(v.abs().max(dim=1).values, min=LEAST)
        return torch.round(v * (127.0 / most).unsqueeze(1)), most / 127.0
    block = torch.arange(k, device=DEVICE) // BLOCK
    most = torch.full((rows, int(block[-1]) + 1), LEAST, device=DEVICE, dtype=torch.float64)
    most = most.scatter_reduce(1, block.expand(rows, -1), v.abs(), "amax")
    return _nearest_e4m3(v * MOST["f8"] / most[:, block]), most / MOST["f8"]


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["op"] == "norm":
        total = s.x.double() + s.residual.double()
        v = total.to(s.x.dtype).double()      # (the sum is stored, and what is stored is what the norm is of)
        y = v / torch.sqrt(v.pow(2).sum(dim=1, keepdim=True) / c["k"] + EPS) * s.weight.double()
        codes, scales = _exact_codes(y, c["codes"])
        return {"sum": total, "y": y, "codes": codes if c["codes"] == "f8" else codes * scales.unsqueeze(1), "scales": scales}
    if c["op"] == "rows":
        v = s.x.double()
        v = _exact_glu(c["act"], v[:, :c["k"]], v[:, c["k"]:]) if c["glu"] else v
        codes, scales = _exact_codes(v, "i8")
        return {"codes": codes * scales.unsqueeze(1) if c["glu"] else None, "scales": scales}
    if c["op"] == "layer":
        T, K, I = c["tokens"], c["top_k"], c["inter"]
        ids, weights = s.ids.long(), s.weights.double()
        if c["routed"]:
            chosen = torch.gather(s.logits.double(), 1, ids)
            weights = torch.softmax(chosen, dim=1)
        out = torch.zeros(T, c["hidden"], device=DEVICE, dtype=torch.float64)
        for e in ids.unique().tolist():
            t, r = (ids == e).nonzero(as_tuple=True)
            g = torch.mm(s.x[t].double(), _exact_matrix(s.w1, s.s1, e).t().contiguous())
            g = g + s.b1[e].double() if s.b1 is not None else g
            y = torch.mm(_exact_glu(c["act"], g[:, :I], g[:, I:]), _exact_matrix(s.w2, s.s2, e).t().contiguous())
            y = y + s.b2[e].double() if s.b2 is not None else y
            out.index_add_(0, t, y * weights[t, r].unsqueeze(1))
        return {"out": out, "ids": None, "weights": weights} if c["routed"] else {"out": out}
    N, k = c["rows"], c["k"]
    b = s.b.double() * s.bs.double().unsqueeze(1)
    out = torch.zeros(s.out.shape, device=DEVICE, dtype=torch.float64)
    ends = [0, c["tokens"]] if c["op"] == "dense" else s.offsets.tolist()
    for e in range(len(ends) - 1):
        lo, hi = ends[e], ends[e + 1]
        if lo == hi:
            continue
        at = s.rows[lo:hi].long() if c["op"] == "grouped" else None
        x = b[at // c["top_k"]] if at is not None and c["gather"] else b[lo:hi]
        y = torch.mm(x, _exact_matrix(s.w, s.ws, e).t().contiguous())
        y = y + s.bias[e].double() if s.bias is not None else y
        if at is None or c["gather"]:
            out[lo:hi] = y
        else:
            out[at] = y
    return {"out": out}
