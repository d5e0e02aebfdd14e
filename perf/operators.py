"""Measured cases of the 8-bit linear path: norm with 8-bit rows, row quantiser, matrix product with a fused epilogue.

`run` computes an operator either in its plain form (elementary torch operations in fp32) or, with `own`, through the
public calls of `dace_onnx_b200.ops`. All tensors live on the GPU; outputs go to buffers that the caller keeps, as in the
framework's own runners.

norm      h = x + residual, y = h / sqrt(mean(h^2) + eps) * gamma; returned as e4m3 codes with one scale a row (or y in x's
          type) and the updated residual h.
quantise  y = x, or act(gate) * x, as e4m3 codes with one scale a row.
product   Y = act((A W^T) * a_scale[m] * w_scale[n] + bias[n]) + residual; A [M, K], W [N, K].

e4m3 rows: a = max(max|y|, 2^-100), scale = a / 448, code = y / scale rounded to e4m3. Rows of codes start at multiples of
16 bytes (the layout in which the quantiser allocates them).
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
EPS = 1e-5
E4M3_MAX = 448.0
TINY = 2.0 ** -100
ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")


def _norm(name, rows, length, dtype, residual=True, codes=True):
    return {"name": name, "op": "norm", "rows": rows, "len": length, "dtype": dtype, "residual": residual, "codes": codes}


def _quantise(name, rows, length, dtype, act="none", gate=False):
    return {"name": name, "op": "quantise", "rows": rows, "len": length, "dtype": dtype, "act": act, "gate": gate}


def _product(name, m, n, k, dtype, out, act="none", bias=False, residual=False):
    return {"name": name, "op": "product", "m": m, "n": n, "k": k, "dtype": dtype, "out": out, "act": act, "bias": bias,
            "residual": residual}


def listed():
    return [
        # the norm in front of a layer when one token is generated: launch latency
        _norm("norm 1 token", 1, 4096, "bf16"),
        # the norm over a long prompt of a wide model: memory bandwidth
        _norm("norm prompt", 8192, 8192, "bf16"),
        # rows of the encoder that the benchmark runs (hidden 1024), fp32 activations
        _norm("norm fp32 rows", 16384, 1024, "f32"),
        # a ragged batch and a width that no vector access divides, output kept in 16 bits
        _norm("norm odd width", 1023, 2561, "f16", codes=False),
        # the gated activation of an MLP for a small batch of single tokens
        _quantise("gate 16 tokens", 16, 14336, "bf16", act="silu", gate=True),
        # the same over a prompt
        _quantise("gate prompt", 8192, 14336, "bf16", act="silu", gate=True),
        # the encoder's widest activations (4096) before its second MLP product
        _quantise("quantise fp32 rows", 16384, 4096, "f32"),
        # attention output projection of one token
        _product("product 1 token", 1, 4096, 4096, "e4m3", "bf16", residual=True),
        # gate and up projections of a batch of 32 single tokens: the weights' bytes
        _product("product 32 tokens", 32, 28672, 4096, "e4m3", "bf16"),
        # odd sizes everywhere, fp32 output, the whole epilogue
        _product("product odd", 333, 1501, 1000, "e4m3", "f32", act="gelu", bias=True, residual=True),
        # a prompt through an up projection
        _product("product prompt", 8192, 14336, 4096, "e4m3", "bf16", act="silu", bias=True),
        # the encoder's first MLP product on 16-bit operands
        _product("product bf16", 16384, 4096, 1024, "bf16", "bf16", act="gelu", bias=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "quantise", "product", "product"))
    if op != "product":
        length = _log(rng, 64, 16384)
        if rng.random() < 0.6:
            length = max(64, length // 64 * 64)
        rows = min(_log(rng, 1, 16384), (1 << 26) // length)
        dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
        if op == "norm":
            c = _norm("", rows, length, dtype, residual=rng.random() < 0.7, codes=rng.random() < 0.7)
        else:
            gate = rng.random() < 0.6
            c = _quantise("", rows, length, dtype, act=rng.choice(ACTS[1:]) if gate else "none", gate=gate)
    else:
        n, k = _log(rng, 64, 16384), _log(rng, 64, 8192)
        if rng.random() < 0.6:
            n, k = max(64, n // 64 * 64), max(64, k // 64 * 64)
        dtype = rng.choice(("e4m3", "e4m3", "bf16", "f16"))
        if dtype != "e4m3":
            k = k // 8 * 8
        m = min(_log(rng, 1, 16384), 8192 * 14336 * 4096 // (n * k))
        out = rng.choice(("bf16", "f16", "f32")) if dtype == "e4m3" else rng.choice((dtype, dtype, "f32"))
        c = _product("", m, n, k, dtype, out, act=rng.choice(ACTS), bias=rng.random() < 0.5, residual=rng.random() < 0.5)
    del c["name"]
    return c


def _row_buffer(rows, length, dtype):
    """[rows, length] whose rows start at multiples of 16 bytes."""
    per = 16 // dtype.itemsize
    return torch.empty(rows, -(-length // per) * per, device="cuda", dtype=dtype)[:, :length]


def _codes_of(rows):
    """What a program that quantised `rows` (fp32) holds: e4m3 codes in padded rows, and scales."""
    scale = rows.abs().amax(1).clamp_min(TINY) / E4M3_MAX
    codes = _row_buffer(rows.shape[0], rows.shape[1], torch.float8_e4m3fn)
    codes.copy_(rows / scale[:, None])
    return codes, scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=torch.float32)  # noqa: E731
    s = dict(case)
    if case["op"] in ("norm", "quantise"):
        rows, length, t = case["rows"], case["len"], TYPES[case["dtype"]]
        # a few channels are larger than the others, as in trained transformers
        channel = torch.where(torch.rand(length, generator=g, device="cuda") < 0.01, 8.0, 1.0)
        s["x"] = (normal(rows, length) * channel).to(t)
        s["codes_out"] = _row_buffer(rows, length, torch.float8_e4m3fn)
        s["scale_out"] = torch.empty(rows, device="cuda", dtype=torch.float32)
        if case["op"] == "norm":
            s["residual_in"] = (normal(rows, length) * 2).to(t) if case["residual"] else None
            s["gamma"] = (1 + 0.1 * normal(length)).to(t)
            s["h_out"] = torch.empty_like(s["x"]) if case["residual"] else None
            s["y_out"] = torch.empty_like(s["x"])
        else:
            s["gate_in"] = (normal(rows, length) * 2).to(t) if case["gate"] else None
        return s
    m, n, k, t = case["m"], case["n"], case["k"], TYPES[case["dtype"]]
    a, w = normal(m, k), normal(n, k) * (1 / math.sqrt(k))
    if case["dtype"] == "e4m3":
        s["a"], s["a_scale"] = _codes_of(a)
        s["w"], s["w_scale"] = _codes_of(w)
    else:
        s["a"], s["w"], s["a_scale"], s["w_scale"] = a.to(t), w.to(t), None, None
    o = TYPES[case["out"]]
    s["bias_in"] = (normal(n) * 0.5).to(o) if case["bias"] else None
    s["residual_in"] = normal(m, n).to(o) if case["residual"] else None
    s["y_out"] = torch.empty(m, n, device="cuda", dtype=o)
    return s


def _act(v, act):
    if act == "relu":
        return torch.maximum(v, torch.zeros((), device=v.device))
    if act == "gelu":
        return v * 0.5 * (1 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return v * 0.5 * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    if act == "silu":
        return v / (1 + torch.exp(-v))
    return v


def _quantised(y):
    scale = y.abs().amax(1).clamp_min(TINY) / E4M3_MAX
    return (y / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale


def _plain(s):
    if s["op"] == "norm":
        h = s["x"].float()
        if s["residual_in"] is not None:
            h = h + s["residual_in"].float()
        y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * s["gamma"].float()
        out = list(_quantised(y)) if s["codes"] else [y.to(s["x"].dtype)]
        return out + ([h.to(s["x"].dtype)] if s["residual_in"] is not None else [])
    if s["op"] == "quantise":
        y = s["x"].float()
        if s["gate_in"] is not None:
            y = _act(s["gate_in"].float(), s["act"]) * y
        return list(_quantised(y))
    y = s["a"].float() @ s["w"].float().t()
    if s["a_scale"] is not None:
        y = y * s["a_scale"][:, None] * s["w_scale"]
    if s["bias_in"] is not None:
        y = y + s["bias_in"].float()
    y = _act(y, s["act"])
    if s["residual_in"] is not None:
        y = y + s["residual_in"].float()
    return [y.to(s["y_out"].dtype)]


def _own(s):
    from dace_onnx_b200 import ops
    if s["op"] == "norm":
        if s["codes"]:
            ops.rmsnorm_quantize(s["x"], s["gamma"], residual=s["residual_in"], eps=EPS, out=s["codes_out"],
                                 scale=s["scale_out"], residual_out=s["h_out"])
            out = [s["codes_out"], s["scale_out"]]
        else:
            ops.rmsnorm(s["x"], s["gamma"], residual=s["residual_in"], eps=EPS, out=s["y_out"], residual_out=s["h_out"])
            out = [s["y_out"]]
        return out + ([s["h_out"]] if s["h_out"] is not None else [])
    if s["op"] == "quantise":
        ops.quantize_rows(s["x"], gate=s["gate_in"], activation=s["act"], out=s["codes_out"], scale=s["scale_out"])
        return [s["codes_out"], s["scale_out"]]
    ops.matmul_scaled(s["a"], s["w"], a_scale=s["a_scale"], w_scale=s["w_scale"], bias=s["bias_in"],
                      activation=s["act"], residual=s["residual_in"], out=s["y_out"])
    return [s["y_out"]]


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    if case["op"] in ("norm", "quantise"):
        n, b = case["rows"] * case["len"], SIZE[case["dtype"]]
        if case["op"] == "norm":
            moved = n * b * (3 if case["residual"] else 1) + case["len"] * b
            moved += n + 4 * case["rows"] if case["codes"] else n * b
        else:
            moved = n * b * (2 if case["gate"] else 1) + n + 4 * case["rows"]
        return {"bytes": moved, "flops": 8 * n}
    m, n, k, b, o = case["m"], case["n"], case["k"], SIZE[case["dtype"]], SIZE[case["out"]]
    moved = (m + n) * k * b + m * n * o * (2 if case["residual"] else 1) + (n * o if case["bias"] else 0)
    moved += 4 * (m + n) if case["dtype"] == "e4m3" else 0
    return {"bytes": moved, "flops": 2 * m * n * k}


def _act64(v, act):
    if act == "none":
        return v
    if act == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if act == "gelu":
        return v * torch.special.ndtr(v)
    if act == "gelu_tanh":
        inner = math.sqrt(2 / math.pi) * v * (1 + 0.044715 * v.square())
        return v * torch.sigmoid(2 * inner)
    return v * torch.sigmoid(v)


def exact(case, seed):
    """The same outputs in 64 bits, before they are rounded to their types."""
    s = prepare(case, seed)
    wide = lambda t: t.to(torch.float64)  # noqa: E731
    rows_of = lambda y: (lambda top: [y * (E4M3_MAX / top)[:, None], top / E4M3_MAX])(  # noqa: E731
        torch.clamp(y.abs().max(dim=1).values, min=TINY))
    if case["op"] == "norm":
        h = wide(s["x"]) if s["residual_in"] is None else wide(s["x"]) + wide(s["residual_in"])
        power = torch.einsum("ij,ij->i", h, h) / case["len"]
        y = wide(s["gamma"])[None] * h / torch.sqrt(power + EPS)[:, None]
        out = rows_of(y) if case["codes"] else [y]
        return out if s["residual_in"] is None else out + [h]
    if case["op"] == "quantise":
        y = wide(s["x"])
        return rows_of(y if s["gate_in"] is None else y * _act64(wide(s["gate_in"]), case["act"]))
    a, w = wide(s["a"]), wide(s["w"])
    if s["a_scale"] is not None:
        a, w = a * wide(s["a_scale"])[:, None], w * wide(s["w_scale"])[:, None]
    y = torch.einsum("mk,nk->mn", a, w)
    del a, w
    y = _act64(y if s["bias_in"] is None else y + wide(s["bias_in"]), case["act"])
    return [y if s["residual_in"] is None else y + wide(s["residual_in"])]
