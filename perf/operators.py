"""The block-scaled FP8 and the grouped products of this engine, as cases that can be timed and checked one by one.

A case is a dict of plain values; `op` names the operator:

- "quantize": rows of activations to e4m3 codes with one fp32 scale per 128 (vbm_quantize_fp8);
- "glu": the gated activation of an expert's gate and up halves, quantized the same way
  (vbm_glu_quantize_fp8);
- "dense": the product of FP8 weights, one scale per 128 x 128 block, with such activations
  (vbm_mul_mat_fp8);
- "grouped": the products of tokens grouped by expert, ragged, with FP8 or 16-bit expert weights
  (vbm_grouped_mul_mat). `gather`: the gate_up side, which reads each token's row for every expert it is
  routed to and writes in grouped order; else the down side, which reads grouped order and writes each
  (token, rank) row to its place.

Where `own` is false, `run` computes the same in elementary torch operations, in 32 bits.
"""
import math
import sys
from pathlib import Path

import torch

own = False
DEVICE = "cuda"
TORCH_TYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPE_ID = {"f32": 0, "f16": 1, "bf16": 30, "f8": 256}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "f8": 1}
SILU, OAI = 0, 1
ALPHA, LIMIT = 1.702, 7.0
BLOCK = 128
MOST = 448.0                # the largest e4m3 value
LEAST = 2.0 ** -116         # blocks whose values are all smaller share this one's scale


def listed():
    return [
        # one token's activations before the FP8 experts of a decode step: latency
        {"name": "quantize_1x2880_f32", "op": "quantize", "rows": 1, "k": 2880, "type": "f32"},
        # the activations of a long prompt
        {"name": "quantize_8192x4096_bf16", "op": "quantize", "rows": 8192, "k": 4096, "type": "bf16"},
        # a decode step between the two expert products: eight experts of one token, fused gate | up rows
        {"name": "glu_8x768_bf16", "op": "glu", "rows": 8, "k": 768, "type": "bf16", "act": SILU},
        # the same in prefill, 2048 tokens to four experts each
        {"name": "glu_8192x2880_f32", "op": "glu", "rows": 8192, "k": 2880, "type": "f32", "act": OAI},
        # a dense projection of one decoded token: the weights are read once
        {"name": "dense_1x5760x2880", "op": "dense", "tokens": 1, "rows": 5760, "k": 2880, "bias": False, "out": "f32"},
        # a short odd-sized prompt, output rows and depth that end inside a block
        {"name": "dense_333x2880x2880", "op": "dense", "tokens": 333, "rows": 2880, "k": 2880, "bias": True, "out": "bf16"},
        # a large prefill batch
        {"name": "dense_4096x4096x4096", "op": "dense", "tokens": 4096, "rows": 4096, "k": 4096, "bias": False, "out": "bf16"},
        # one decoded token through the gate_up of eight FP8 experts
        {"name": "grouped_f8_1", "op": "grouped", "type": "f8", "tokens": 1, "top_k": 8, "experts": 128, "rows": 1536, "k": 2048,
         "gather": True, "bias": False, "masked": False, "out": "bf16"},
        # a decode batch: some rows for each of 32 FP8 experts, with biases
        {"name": "grouped_f8_64", "op": "grouped", "type": "f8", "tokens": 64, "top_k": 4, "experts": 32, "rows": 5760, "k": 2880,
         "gather": True, "bias": True, "masked": False, "out": "f32"},
        # prefill of 2048 tokens over 128 FP8 experts, some routes masked
        {"name": "grouped_f8_2048", "op": "grouped", "type": "f8", "tokens": 2048, "top_k": 8, "experts": 128, "rows": 1536, "k": 2048,
         "gather": True, "bias": False, "masked": True, "out": "bf16"},
        # a decode batch over 16-bit experts, the down side
        {"name": "grouped_bf16_16", "op": "grouped", "type": "bf16", "tokens": 16, "top_k": 4, "experts": 32, "rows": 2880, "k": 2880,
         "gather": False, "bias": True, "masked": False, "out": "f32"},
        # prefill of an odd-sized prompt over 16-bit experts, the down side
        {"name": "grouped_f16_1517", "op": "grouped", "type": "f16", "tokens": 1517, "top_k": 6, "experts": 64, "rows": 2048, "k": 1408,
         "gather": False, "bias": False, "masked": True, "out": "f32"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["quantize", "glu", "dense", "dense", "grouped", "grouped", "grouped", "grouped"])
    out = rng.choice(["f32", "bf16", "f16"])
    if op in ("quantize", "glu"):
        k, rows = 16 * _log_int(rng, 4, 512), _log_int(rng, 1, 16384)
        rows = max(1, min(rows, 8192 * (2880 if op == "glu" else 4096) // k))
        c = {"op": op, "rows": rows, "k": k, "type": out}
        return {**c, "act": rng.choice([SILU, OAI])} if op == "glu" else c
    # row counts that are no multiple of anything now and then; depths are multiples of 16 values
    rows = rng.choice([_log_int(rng, 64, 6144), 64 * _log_int(rng, 1, 90)])
    k = 16 * _log_int(rng, 8, 400)
    if op == "dense":
        tokens = _log_int(rng, 1, 4096)
        c = {"op": op, "tokens": tokens, "rows": rows, "k": k, "bias": rng.random() < 0.5, "out": out}
        while 2.0 * c["tokens"] * rows * k > 1.3e11:
            c["tokens"] = c["tokens"] * 2 // 3
        return c
    kind = rng.choice(["f8", "f8", "bf16", "f16"])
    experts = _log_int(rng, 4, 128)
    c = {"op": op, "type": kind, "tokens": _log_int(rng, 1, 2048), "top_k": rng.randint(1, min(8, experts)), "experts": experts,
         "rows": rows, "k": k, "gather": rng.random() < 0.5, "bias": rng.random() < 0.5, "masked": rng.random() < 0.5,
         "out": out}
    # no more weights and products than the listed ones
    while c["experts"] > c["top_k"] and 1.0 * c["experts"] * rows * k > 4.0e8:
        c["experts"] = max(c["top_k"], c["experts"] * 2 // 3)
    while c["tokens"] > 1 and 2.0 * c["tokens"] * c["top_k"] * rows * k > 1.0e11:
        c["tokens"] = c["tokens"] * 2 // 3
    return c


# ------------------------------------------------------------------------------------------ inputs
def _gen(seed, place):
    g = torch.Generator(device=DEVICE)
    g.manual_seed((seed * 1000003 + place * 7919 + 17) & 0x7FFFFFFFFFFF)
    return g


def _normal(seed, place, *shape, std=1.0):
    return torch.randn(*shape, generator=_gen(seed, place), device=DEVICE, dtype=torch.float32) * std


def _activations(seed, place, rows, k):
    """N(0, 1) with a few channels that are ten times as large, as hidden states have them."""
    channel = 1.0 + 9.0 * (torch.rand(k, generator=_gen(seed, place + 1), device=DEVICE) < 0.01)
    return _normal(seed, place, rows, k) * channel


def _fp8_weights(seed, place, experts, rows, k):
    """e4m3 codes [experts][rows][k] (as bytes) and scales [experts][ceil(rows / 128)][ceil(k / 128)] of normal weights."""
    nb, kb = -(-rows // BLOCK), -(-k // BLOCK)
    w = torch.zeros(experts, nb * BLOCK, kb * BLOCK, device=DEVICE)
    w[:, :rows, :k] = _normal(seed, place, experts, rows, k, std=1.0 / math.sqrt(k))
    blocks = w.view(experts, nb, BLOCK, kb, BLOCK)
    scales = blocks.abs().amax(dim=(2, 4)).clamp_(min=LEAST) / MOST
    blocks /= scales[:, :, None, :, None]
    codes = w[:, :rows, :k].to(torch.float8_e4m3fn).view(torch.uint8).contiguous()
    return codes, scales


def _quantize(x):
    """(codes [rows][k] as bytes, scales [rows][ceil(k / 128)]) of fp32 rows."""
    rows, k = x.shape
    kb = -(-k // BLOCK)
    v = torch.nn.functional.pad(x, (0, kb * BLOCK - k)).view(rows, kb, BLOCK)
    most = v.abs().amax(dim=2).clamp_(min=LEAST)
    codes = (v * MOST / most[:, :, None]).clamp_(-MOST, MOST).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8).view(rows, kb * BLOCK)[:, :k].contiguous(), most / MOST


def _routes(c, seed):
    """Routing of the tokens, grouped by expert: offsets [experts + 1] and the (token, rank) rows in grouped order,
    both int32, and what a plain program has to know on the host. Experts are liked unequally; a masked route has none."""
    T, K, E = c["tokens"], c["top_k"], c["experts"]
    score = torch.rand(T, E, generator=_gen(seed, 30), device=DEVICE) + 0.05 * torch.rand(E, generator=_gen(seed, 31), device=DEVICE)
    ids = score.topk(K, dim=1).indices.reshape(-1)
    if c["masked"]:
        ids = torch.where(torch.rand(T * K, generator=_gen(seed, 32), device=DEVICE) < 0.03, torch.full_like(ids, E), ids)
    rows = torch.sort(ids, stable=True).indices.to(torch.int32)
    counts = torch.bincount(ids, minlength=E + 1)[:E]
    offsets = torch.zeros(E + 1, device=DEVICE, dtype=torch.int32)
    offsets[1:] = counts.cumsum(0)
    return offsets, rows, counts


class _State:
    pass


def prepare(case, seed):
    c, s = case, _State()
    s.case = c
    if c["op"] == "quantize":
        s.x = _activations(seed, 1, c["rows"], c["k"]).to(TORCH_TYPE[c["type"]])
    elif c["op"] == "glu":
        # the fused product's rows: gate in the first half of each, up in the second
        s.x = _activations(seed, 1, c["rows"], 2 * c["k"]).to(TORCH_TYPE[c["type"]])
    if c["op"] in ("quantize", "glu"):
        s.codes = torch.empty(c["rows"], c["k"], device=DEVICE, dtype=torch.uint8)
        s.scales = torch.empty(c["rows"], -(-c["k"] // BLOCK), device=DEVICE)
        return s
    grouped = c["op"] == "grouped"
    E, N, k, kind = c.get("experts", 1), c["rows"], c["k"], c.get("type", "f8")
    s.ws = s.bs = None
    if kind == "f8":
        s.w, s.ws = _fp8_weights(seed, 10, E, N, k)
    else:
        s.w = _normal(seed, 10, E, N, k, std=1.0 / math.sqrt(k)).to(TORCH_TYPE[kind])
    s.bias = _normal(seed, 20, E, N, std=0.02) if c["bias"] else None
    entries = c["tokens"] * c.get("top_k", 1)
    b = _activations(seed, 1, c["tokens"] if not grouped or c["gather"] else entries, k)
    if kind == "f8":
        s.b, s.bs = _quantize(b)
    else:
        s.b = b.to(TORCH_TYPE[kind])
    s.out = torch.zeros(entries, N, device=DEVICE, dtype=TORCH_TYPE[c["out"]])
    if grouped:
        s.offsets, s.rows, counts = _routes(c, seed)
        s.used, s.most, s.active = int(counts.sum()), int(counts.max()), counts.nonzero().squeeze(1)
    return s


# --------------------------------------------------------------------------------- the plain forms
def _scaled_weights(w, ws):
    """fp32 weights [experts][rows][k] of codes and block scales."""
    E, N, k = w.shape
    v = w.view(torch.float8_e4m3fn).float()
    by_k = ws.repeat_interleave(BLOCK, dim=2)[:, :, :k]
    whole = N // BLOCK * BLOCK
    if whole:
        v[:, :whole].unflatten(1, (-1, BLOCK)).mul_(by_k[:, :whole // BLOCK, None, :])
    if whole < N:
        v[:, whole:].mul_(by_k[:, -1:, :])
    return v


def _scaled_rows(b, bs):
    return b.view(torch.float8_e4m3fn).float() * bs.repeat_interleave(BLOCK, dim=1)[:, :b.shape[1]]


def _gated(c, x):
    g, u = x[:, :c["k"]].float(), x[:, c["k"]:].float()
    if c["act"] == OAI:
        g, u = g.clamp(max=LIMIT), u.clamp(-LIMIT, LIMIT)
        return g / (1 + torch.exp(-ALPHA * g)) * (u + 1)
    return g / (1 + torch.exp(-g)) * u


def _plain(s):
    c = s.case
    if c["op"] in ("quantize", "glu"):
        codes, scales = _quantize(s.x.float() if c["op"] == "quantize" else _gated(c, s.x))
        return {"codes": codes.view(torch.float8_e4m3fn), "scales": scales}
    if c["op"] == "dense":
        y = _scaled_rows(s.b, s.bs) @ _scaled_weights(s.w, s.ws)[0].T
        if s.bias is not None:
            y += s.bias
        return {"out": y.to(TORCH_TYPE[c["out"]])}
    # the touched experts' rows side by side, padded to the longest, and one batched product
    k = c["k"]
    counts = s.offsets.diff()
    at = torch.arange(s.used, device=DEVICE, dtype=torch.int32)
    expert = torch.searchsorted(s.offsets[1:], at, right=True)
    slot, place = ((counts > 0).cumsum(0) - 1)[expert], at - s.offsets[expert]
    w = s.w[s.active]
    w, b = (_scaled_weights(w, s.ws[s.active]), _scaled_rows(s.b, s.bs)) if s.ws is not None else (w.float(), s.b.float())
    rows = s.rows[:s.used]
    x = torch.zeros(len(s.active), s.most, k, device=DEVICE)
    x[slot, place] = b[rows // c["top_k"]] if c["gather"] else b[:s.used]
    y = torch.bmm(w, x.transpose(1, 2).contiguous())[slot, :, place]
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


def _kernels(s):
    vb, c = _engine(), s.case
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] in ("quantize", "glu"):
        kind = TYPE_ID[c["type"]]
        if c["op"] == "quantize":
            vb.call("vbm_quantize_fp8", kind, s.x.data_ptr(), c["rows"], c["k"], c["k"], s.codes.data_ptr(), s.scales.data_ptr(), stream)
        else:
            x = s.x.data_ptr()
            vb.call("vbm_glu_quantize_fp8", c["act"], kind, x, x + c["k"] * BYTES[c["type"]], c["rows"], c["k"], 2 * c["k"], 2 * c["k"],
                    ALPHA, LIMIT, s.codes.data_ptr(), s.scales.data_ptr(), stream)
        return {"codes": s.codes.view(torch.float8_e4m3fn), "scales": s.scales}
    w = vb.Weights(TYPE_ID[c.get("type", "f8")], s.w.data_ptr(), s.ws.data_ptr() if s.ws is not None else None,
                   s.bias.data_ptr() if s.bias is not None else None, s.w.shape[0], c["rows"], c["k"])
    bs, out = s.bs.data_ptr() if s.bs is not None else None, TYPE_ID[c["out"]]
    if c["op"] == "dense":
        vb.call("vbm_mul_mat_fp8", w, s.b.data_ptr(), bs, c["tokens"], out, s.out.data_ptr(), stream)
    else:
        rows, gather, n = s.rows.data_ptr(), c["gather"], s.out.shape[0]
        vb.call("vbm_grouped_mul_mat", w, s.b.data_ptr(), bs, s.b.shape[0], rows if gather else None, c["top_k"] if gather else 1,
                s.offsets.data_ptr(), n, None if gather else rows, n, out, s.out.data_ptr(), stream)
    return {"out": s.out}


def run(s):
    return _kernels(s) if own else _plain(s)


def work(case):
    c = case
    k = c["k"]
    if c["op"] in ("quantize", "glu"):
        halves = 2 if c["op"] == "glu" else 1
        return {"bytes": c["rows"] * (k * (halves * BYTES[c["type"]] + 1) + 4.0 * -(-k // BLOCK)), "flops": c["rows"] * k * (12.0 if halves == 2 else 3.0)}
    kind, N, E = c.get("type", "f8"), c["rows"], c.get("experts", 1)
    entries = c["tokens"] * c.get("top_k", 1) * (0.97 if c.get("masked") else 1.0)
    touched = E * (1 - (1 - c["top_k"] / E) ** c["tokens"]) if c["op"] == "grouped" else 1
    n_b = c["tokens"] if c["op"] == "dense" or c["gather"] else entries
    scale_bytes = 4.0 * -(-k // BLOCK) * (touched * -(-N // BLOCK) + n_b) if kind == "f8" else 0.0
    lists = 4.0 * (entries + E + 1) if c["op"] == "grouped" else 0.0
    return {"bytes": (touched * N + n_b) * k * BYTES[kind] + scale_bytes + lists + (4.0 * touched * N if c["bias"] else 0) + entries * N * BYTES[c["out"]],
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


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["op"] in ("quantize", "glu"):
        v = s.x.double()
        if c["op"] == "glu":
            g, u = v[:, :c["k"]], v[:, c["k"]:]
            if c["act"] == OAI:
                g, u = torch.clamp(g, max=LIMIT), torch.clamp(u, -LIMIT, LIMIT)
                v = g * torch.sigmoid(ALPHA * g) * (1 + u)
            else:
                v = g * torch.sigmoid(g) * u
        block = torch.arange(c["k"], device=DEVICE) // BLOCK
        most = torch.full((c["rows"], int(block[-1]) + 1), LEAST, device=DEVICE, dtype=torch.float64)
        most = most.scatter_reduce(1, block.expand(c["rows"], -1), v.abs(), "amax")
        return {"codes": _nearest_e4m3(v * MOST / most[:, block]), "scales": most / MOST}
    N, k = c["rows"], c["k"]
    b = s.b.double() if s.bs is None else _e4m3_values(s.b) * _expand(s.bs, 1, k)
    out = torch.zeros(s.out.shape, device=DEVICE, dtype=torch.float64)
    ends = [0, c["tokens"]] if c["op"] == "dense" else s.offsets.tolist()
    for e in range(len(ends) - 1):
        lo, hi = ends[e], ends[e + 1]
        if lo == hi:
            continue
        w = s.w[e].double() if s.ws is None else _e4m3_values(s.w[e]) * _expand(_expand(s.ws[e], 0, N), 1, k)
        at = s.rows[lo:hi].long() if c["op"] == "grouped" else None
        x = b[at // c["top_k"]] if at is not None and c["gather"] else b[lo:hi]
        y = torch.mm(x, w.t().contiguous())
        y = y + s.bias[e].double() if s.bias is not None else y
        if at is None or c["gather"]:
            out[lo:hi] = y
        else:
            out[at] = y
    return {"out": out}
