"""The operators of a decoder layer's dense part in 8 bits, as timed cases.

Four kinds of pass, each the call that a serving program makes of it:

* ``norm`` -- the residual stream gets a block's output added and is normalised
  for the next block, whose input leaves in 8 bits with scales: integers with
  a scale a row, or E4M3 with a scale a row or for every 128 channels; where
  the next block wants them (a router), the normalised rows too.
* ``quant`` -- rows to 8-bit integers with a scale a row, as what feeds a
  product but comes from no norm (attention's output).
* ``linear`` -- the product of such rows with a matrix of 8-bit integers that
  has a scale for each output channel, with bias and residual where a layer
  has them; from rows that are not quantized yet, or from those that are.
* ``ffn`` -- a gated feed-forward block on such matrices: both projections,
  activation and product, the hidden rows to 8 bits, the projection back, the
  residual's addition.

With T the type of the rows, every ``fl`` a rounding to 32 bits:

  norm    h = T(x + residual), g = fl(offset + weight), u = fl(h g),
          y = u / sqrt(mean(h^2) + eps)
  scales  integers: s = fl(max(fl(max |y|), 1e-12) / 127), codes round(y / s);
          E4M3: s = fl(max(fl(max |y|), 1e-10) fl(1 / 448)), codes the E4M3 number
          nearest y / s; ties to even
  linear  T(sum(codes codes) s_row s_channel + bias + residual)
  ffn     a = T(act(gate) up) of the two products, act(z) = z / (1 + exp(-z))
          or gelu in its tanh form; then linear of a's codes

What is held in 8 bits is returned as the values it stands for.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6
# (hidden, intermediate) of the drawn layers
LAYERS = [(1024, 2816), (2048, 5632), (2048, 768), (4096, 11008), (2560, 6912), (512, 1376), (1536, 4096), (5120, 8192)]


def _norm(name, rows, width, *, quant, dtype="bf16", residual=True, keep=False, offset=0.0, spread=1):
    return {"name": name, "kind": "norm", "rows": rows, "width": width, "quant": quant, "dtype": dtype,
            "residual": residual, "keep": keep, "offset": offset, "spread": spread}


def _quant(name, rows, width, *, dtype="bf16", spread=1):
    return {"name": name, "kind": "quant", "rows": rows, "width": width, "dtype": dtype, "spread": spread}


def _linear(name, rows, k, n, *, dtype="bf16", given=False, bias=False, residual=False, spread=1):
    return {"name": name, "kind": "linear", "rows": rows, "width": k, "out": n, "dtype": dtype, "given": given,
            "bias": bias, "residual": residual, "spread": spread}


def _ffn(name, rows, width, inter, *, dtype="bf16", act="silu", given=False, residual=True, spread=1):
    return {"name": name, "kind": "ffn", "rows": rows, "width": width, "inter": inter, "dtype": dtype, "act": act,
            "given": given, "residual": residual, "spread": spread}


def listed():
    return [
        # one token between attention and feed-forward: latency alone
        _norm("norm-1", 1, 2048, quant="int8"),
        # a long prompt's rows at the same place
        _norm("norm-8192", 8192, 4096, quant="int8"),
        # before a mixture of experts: rows for the router, E4M3 groups for the experts; a gain of 1 + weight
        _norm("norm-777-moe", 777, 2048, quant="fp8-128", dtype="f16", keep=True, offset=1.0),
        # attention's output of a decode step of some streams
        _quant("quant-13", 13, 8192),
        # rows of an odd width
        _quant("quant-5003-odd", 5003, 2501, dtype="f16"),
        # one token through the joint query, key and value projection
        _linear("linear-1", 1, 2048, 2560),
        # a decode step of some streams through the output projection, rows in 8 bits already
        _linear("linear-13", 13, 4096, 4096, given=True, residual=True),
        # a short prompt, an odd number of channels, bias
        _linear("linear-509", 509, 2048, 5003, dtype="f16", bias=True),
        # a long prompt
        _linear("linear-8192", 8192, 4096, 4096, given=True),
        # one token through a whole feed-forward block
        _ffn("ffn-1", 1, 2048, 5632),
        # a decode step of many streams, the other activation, fp16
        _ffn("ffn-47", 47, 4096, 11008, dtype="f16", act="gelu_tanh"),
        # a long prompt behind a norm that gave its rows in 8 bits
        _ffn("ffn-4096", 4096, 4096, 12288, given=True),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "quant", "linear", "linear", "ffn", "ffn"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"] if kind in ("norm", "quant") else ["bf16", "bf16", "f16"])
    spread = rng.randrange(1000)
    hidden, inter = rng.choice(LAYERS)
    if kind in ("norm", "quant"):
        width = hidden if rng.random() < 0.5 else _log_int(rng, 33, 8192)
        rows = min(_log_int(rng, 1, 8192), (1 << 24) // width)
        if kind == "quant":
            return _unnamed(_quant("", rows, width, dtype=dtype, spread=spread))
        quant = rng.choice(["int8", "int8", "fp8", "fp8-128"])
        if quant == "fp8-128":
            width = max(128, width // 128 * 128)
        return _unnamed(_norm("", rows, width, quant=quant, dtype=dtype, residual=rng.random() < 0.7,
                              keep=rng.random() < 0.4, offset=rng.choice([0.0, 1.0]), spread=spread))
    if kind == "linear":
        k, n = rng.choice([(hidden, inter), (inter, hidden), (hidden, hidden), (_log_int(rng, 65, 6000), _log_int(rng, 33, 9000))])
        given = k % 16 == 0 and rng.random() < 0.4
        return _unnamed(_linear("", _log_int(rng, 1, 6000), k, n, dtype=dtype, given=given, bias=rng.random() < 0.3,
                                residual=rng.random() < 0.4, spread=spread))
    return _unnamed(_ffn("", _log_int(rng, 1, 3000), hidden, inter, dtype=dtype, act=rng.choice(["silu", "silu", "gelu_tanh"]),
                         given=rng.random() < 0.4, residual=rng.random() < 0.6, spread=spread))


def _unnamed(case):
    return {k: v for k, v in case.items() if k != "name"}


def work(case):
    rows, width, size = case["rows"], case["width"], DTYPES[case["dtype"]].itemsize
    cells = rows * width
    if case["kind"] == "quant":  # rows in, codes out; codes in, values out
        return {"bytes": 2 * cells * size + 2 * cells + 8 * rows, "flops": 4 * cells}
    if case["kind"] == "norm":
        scales = rows * (width // 128 if case["quant"] == "fp8-128" else 1)
        moved = cells * (2 * size if case["residual"] else 0) + cells * size  # residual in and out, x in
        moved += cells * size if case["keep"] else 0
        return {"bytes": moved + width * size + 2 * (cells + 4 * scales) + cells * size, "flops": 8 * cells}
    first = cells + 4 * rows if case["given"] else cells * size
    if case["kind"] == "linear":
        k, n = width, case["out"]
        return {"bytes": first + n * (k + 4) + rows * n * size * (2 if case["residual"] else 1) + (4 * n if case["bias"] else 0),
                "flops": 2 * rows * n * k}
    inter = case["inter"]
    return {"bytes": first + 3 * inter * width + 4 * (2 * inter + width) + cells * size * (2 if case["residual"] else 1),
            "flops": 6 * rows * inter * width}


# --------------------------------------------------------------------- inputs

def _stream(rows, width, dtype, g, device, size):
    """Rows of a residual stream: normal values, some channels far larger, rows of different size."""
    x = torch.randn(rows, width, generator=g, device=device)
    loud = 1 + 15 * (torch.rand(width, generator=g, device=device) < 0.01).float()
    each = size * torch.exp(0.4 * torch.randn(rows, 1, generator=g, device=device))
    return (x * loud * each).to(dtype)


def _matrix(n, k, g, device):
    """(codes [n, k], scales [n]) of a matrix, its rows in storage that is whole 16 bytes a row."""
    held = torch.zeros(n, -(-k // 16) * 16, dtype=torch.int8, device=device)
    for part in held.split(8192):
        part[:, :k] = (torch.randn(part.shape[0], k, generator=g, device=device) * 33).round().clamp(-127, 127).to(torch.int8)
    scales = torch.exp(0.25 * torch.randn(n, generator=g, device=device)) * (k ** -0.5 / 33)
    return held[:, :k], scales


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(int(seed) * 1009 + case["spread"])
    dtype, rows, width = DTYPES[case["dtype"]], case["rows"], case["width"]
    state = {"case": case}
    if case["kind"] == "norm":
        state["x"] = _stream(rows, width, dtype, g, device, 0.6)
        state["weight"] = (0.1 * torch.randn(width, generator=g, device=device) + 1 - case["offset"]).to(dtype)
        state["residual"] = _stream(rows, width, dtype, g, device, 1.7) if case["residual"] else None
        return state
    if case["kind"] == "quant":
        state["x"] = _stream(rows, width, dtype, g, device, 0.4)
        return state
    if case["given"]:  # as a norm's output holds them
        x = _stream(rows, width, torch.float32, g, device, 1.0)
        state["scales"] = x.abs().amax(-1) / 127
        state["codes"] = (x / state["scales"][:, None]).round().clamp(-127, 127).to(torch.int8)
    else:
        state["x"] = _stream(rows, width, dtype, g, device, 1.0)
    if case["kind"] == "linear":
        state["w"], state["w_scales"] = _matrix(case["out"], width, g, device)
        state["bias"] = torch.randn(case["out"], generator=g, device=device) if case["bias"] else None
    else:  # gate rows, then up rows, as a checkpoint's joint matrix has them
        state["w"], state["w_scales"] = _matrix(2 * case["inter"], width, g, device)
        state["back"], state["back_scales"] = _matrix(width, case["inter"], g, device)
    state["residual"] = None
    if case["residual"]:
        state["residual"] = _stream(rows, case["out"] if case["kind"] == "linear" else width, dtype, g, device, 1.0)
    return state


# ------------------------------------------------------------------ plain form

def _int8(y):
    """(codes, scales) of rows: borders between codes in 64 bits."""
    scales = y.abs().amax(-1, keepdim=True).float().clamp(min=1e-12) / 127
    return (y.double() / scales.double()).round().clamp(-127, 127).float(), scales


def _e4m3(y, group):
    """(values of the codes, scales) of each ``group`` channels.  64 bits go to 32 so that no value falls onto a border
    that it is not on."""
    y = y.unflatten(-1, (-1, group))
    scales = y.abs().amax(-1, keepdim=True).float().clamp(min=1e-10) * torch.tensor(1 / 448, dtype=torch.float32).item()
    exact = (y / scales.double()).clamp(-448, 448)
    grid = torch.exp2(torch.frexp(exact).exponent.clamp(min=-5).double() - 4)
    return ((exact / grid).round() * grid).float(), scales


def _plain_norm(state):
    case = state["case"]
    x, residual = state["x"], state["residual"]
    dtype = x.dtype
    h = x if residual is None else (x.float() + residual.float()).to(dtype)
    gain = state["weight"].float() + case["offset"]
    by = torch.rsqrt(h.double().square().mean(-1, keepdim=True) + EPS)
    y = (h.float() * gain).double() * by
    if case["quant"] == "int8":
        codes, scales = _int8(y)
        held = codes * scales
    else:
        codes, scales = _e4m3(y, case["width"] if case["quant"] == "fp8" else 128)
        held = (codes * scales).flatten(-2)
    out = {"held": held.to(dtype)}
    if residual is not None:
        out["h"] = h
    if case["keep"]:
        out["y"] = y.float().to(dtype)
    return out


def _plain_product(codes, scales, w, w_scales):
    return codes @ w.float().T * w_scales * scales


def _plain_rows(state):
    if state["case"]["given"]:
        return state["codes"].float(), state["scales"][:, None]
    return _int8(state["x"])


def _plain_linear(state):
    out = _plain_product(*_plain_rows(state), state["w"], state["w_scales"])
    if state["bias"] is not None:
        out = out + state["bias"]
    if state["residual"] is not None:
        out = out + state["residual"].float()
    return out.to(DTYPES[state["case"]["dtype"]])


def _plain_ffn(state):
    case = state["case"]
    dtype = DTYPES[case["dtype"]]
    gate, up = _plain_product(*_plain_rows(state), state["w"], state["w_scales"]).chunk(2, -1)
    if case["act"] == "silu":
        gate = gate / (1 + torch.exp(-gate))
    else:
        gate = gate / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (gate + 0.044715 * gate * gate * gate)))
    out = _plain_product(*_int8((gate * up).to(dtype)), state["back"], state["back_scales"])
    if state["residual"] is not None:
        out = out + state["residual"].float()
    return out.to(dtype)


# ------------------------------------------------------------------------ runs

def _own(state):
    """The same passes through the framework's operators."""
    import os
    import sys

    place = os.path.abspath("drama3-studio_amd")
    if place not in sys.path:
        sys.path.insert(0, place)
    from drama_moe.int8 import Int8Weight, QuantRows, int8_feed_forward, int8_linear, quantize_rows
    from drama_moe.norm import rms_norm

    case = state["case"]
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "norm":
        made = rms_norm(state["x"], state["weight"], residual=state["residual"], eps=EPS, offset=case["offset"],
                        quant=case["quant"], rows=case["keep"])
        out = {"held": made.quant.dequantize(dtype)}
        if case["residual"]:
            out["h"] = made.hidden
        if case["keep"]:
            out["y"] = made.rows
        return out
    if case["kind"] == "quant":
        return quantize_rows(state["x"]).dequantize(dtype)
    x = QuantRows(state["codes"], state["scales"]) if case["given"] else state["x"]
    weight = Int8Weight(state["w"], state["w_scales"])
    if case["kind"] == "linear":
        return int8_linear(x, weight, bias=state["bias"], residual=state["residual"], dtype=dtype)
    return int8_feed_forward(x, weight, Int8Weight(state["back"], state["back_scales"]), activation=case["act"],
                             residual=state["residual"], dtype=dtype)


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind == "norm":
        return _plain_norm(state)
    if kind == "quant":
        codes, scales = _int8(state["x"])
        return (codes * scales).to(state["x"].dtype)
    return _plain_linear(state) if kind == "linear" else _plain_ffn(state)


# ----------------------------------------------------------------------- exact

def _nearest_int8(v):
    """Codes and scales of rows in 64 bits, by the definition: the floor half a step up, or the even one of a tie's two."""
    top = torch.linalg.vector_norm(v, math.inf, -1, keepdim=True).float()
    step = (torch.maximum(top, torch.full_like(top, 1e-12)) / 127).double()
    ratio = v / step
    code = torch.floor(ratio + 0.5)
    code = torch.where((code - ratio == 0.5) & (code.long() % 2 != 0), code - 1, code)
    return code.clamp(-127, 127), step


def _nearest_e4m3(v, group):
    """Values of the nearest E4M3 numbers, looked up among all of them."""
    table = torch.arange(127, dtype=torch.uint8, device=v.device).view(torch.float8_e4m3fn).double()
    middle = (table[1:] + table[:-1]) / 2
    v = v.view(v.shape[0], -1, group)
    top = torch.linalg.vector_norm(v, math.inf, -1, keepdim=True).float()
    step = (torch.maximum(top, torch.full_like(top, 1e-10)) * torch.tensor(1 / 448, dtype=torch.float32).item()).double()
    size = (v / step).abs()
    low = torch.searchsorted(middle, size.contiguous(), right=False)
    high = torch.searchsorted(middle, size.contiguous(), right=True)
    at = torch.where((low != high) & (low % 2 == 1), high, low)  # on a border: the even one
    return torch.copysign(table[at], v) * step


def _sums(codes, w):
    """The integer sums of codes [M, K] and w [N, K], in 64 bits."""
    return torch.cat([torch.mm(part, w.double().t()) for part in codes.double().split(2048)])


def exact(case, seed):
    state = prepare(case, seed)
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "norm":
        parts = []
        weight = (state["weight"].double() + case["offset"]).float().double()
        residual = state["residual"]
        for at in range(0, case["rows"], 1024):
            h = state["x"][at:at + 1024].double()
            if residual is not None:
                h = (h + residual[at:at + 1024].double()).to(dtype).double()
            u = (h * weight).float().double()
            y = u / torch.sqrt(torch.sum(h * h, -1, keepdim=True) / case["width"] + EPS)
            if case["quant"] == "int8":
                code, step = _nearest_int8(y)
                held = code * step
            else:
                held = _nearest_e4m3(y, case["width"] if case["quant"] == "fp8" else 128).reshape(y.shape)
            parts.append({"held": held, "h": h, "y": y})
        names = ["held"] + (["h"] if residual is not None else []) + (["y"] if case["keep"] else [])
        return {name: torch.cat([p[name] for p in parts]) for name in names}
    if case["kind"] == "quant":
        parts = [_nearest_int8(x.double()) for x in state["x"].split(1024)]
        return torch.cat([code * step for code, step in parts])
    if case["given"]:
        codes, step = state["codes"].double(), state["scales"].double().unsqueeze(1)
    else:
        codes, step = _nearest_int8(state["x"].double())
    first = _sums(codes, state["w"]).mul_(step).mul_(state["w_scales"].double())
    if case["kind"] == "linear":
        if state["bias"] is not None:
            first += state["bias"].double()
        return first if state["residual"] is None else first + state["residual"].double()
    inter = case["inter"]
    gate, up = first[:, :inter], first[:, inter:]
    if case["act"] == "silu":
        gate = gate * torch.sigmoid(gate)
    else:
        gate = 0.5 * gate * (1 + torch.tanh(math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3)))
    hidden = torch.mul(gate, up).to(dtype).double()  # the hidden rows are of the rows' type
    codes, step = _nearest_int8(hidden)
    out = _sums(codes, state["back"]).mul_(step).mul_(state["back_scales"].double())
    return out if state["residual"] is None else out + state["residual"].double()
