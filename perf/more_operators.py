"""The measured workloads of the microscaling operators and the norm that feeds them, through their public entry points.

Four kinds of call around the quantised linears of a decoder layer: the residual's addition with its root-mean-square
norm, writing floats or the 8-bit (and 4-bit) rows that the next linear takes; quantising to microscaling blocks (32
elements of 4-bit or 8-bit floating point under one power of two) and reading them back; linears over weights of 4-bit
blocks; and the gated product of a feed-forward block over two such weights, ready for the next linear.  Shapes are
TinyLlama-1.1B's (2048, 5632), Llama-7B class (4096, 11008) and Llama-3-8B's (4096, 14336), and generic ones; ``draw``
spreads more cases over the same ranges.

With ``own`` false everything is plain torch in 32 bits, rounded once at the end; the sum of squares is in 64 bits, since
codes next to a rounding border go by its last bits.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_PACKAGE = str(Path(__file__).resolve().parent.parent / "qpu-xla-triton_amd")
_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_SIZE = {"float32": 4.0, "bfloat16": 2.0, "float16": 2.0, "mxfp8": 33 / 32, "mxfp4": 17 / 32, "int8": 1.0, "q8_0": 34 / 32}
BLOCK = 32
EPSILON = 1e-5
# A drawn case costs no more than the largest listed ones.
MOST_FLOPS = 4 * 4096 * 4096 * 14336
MOST_BYTES = 700_000_000


def listed():
    return [
        # One token of a TinyLlama-1.1B stream, fp32 from the linears, ready for a microscaling linear. Latency.
        {"name": "norm_t1_mxfp8", "kind": "norm", "tokens": 1, "width": 2048, "input": "float32", "residual": "float32",
         "output": "mxfp8"},
        # A prefill chunk of a Llama-7B class model before a W8A8 linear: the ordinary large call.
        {"name": "norm_t4096_int8", "kind": "norm", "tokens": 4096, "width": 4096, "input": "bfloat16",
         "residual": "bfloat16", "output": "int8"},
        # A ragged batch whose norm stays in floats.
        {"name": "norm_t777_half", "kind": "norm", "tokens": 777, "width": 11008, "input": "float16",
         "residual": "float16", "output": "float16"},
        # A Llama-3-8B feed-forward weight quantised at load time, and read back.
        {"name": "quantize_weight_mxfp4", "kind": "quantize", "rows": 14336, "columns": 4096, "input": "bfloat16",
         "format": "mxfp4", "output": "bfloat16"},
        # fp32 activations of a batch, quantised and read back.
        {"name": "quantize_rows_mxfp8", "kind": "quantize", "rows": 509, "columns": 11008, "input": "float32",
         "format": "mxfp8", "output": "float32"},
        # One token through a TinyLlama-1.1B feed-forward linear, fp32 as its other linears. Latency.
        {"name": "linear_decode_m1", "kind": "linear", "rows": 1, "columns": 2048, "outputs": 5632, "input": "float32",
         "format": "mxfp8", "output": "float32", "bias": False},
        # A serving batch of eight through a Llama-3-8B linear: bound by the weight's bytes.
        {"name": "linear_decode_m8", "kind": "linear", "rows": 8, "columns": 4096, "outputs": 14336, "input": "bfloat16",
         "format": "mxfp8", "output": "bfloat16", "bias": False},
        # A ragged batch between decode and prefill, the long way down, from rows that the norm quantised.
        {"name": "linear_m77_mxfp4", "kind": "linear", "rows": 77, "columns": 11008, "outputs": 4096, "input": "mxfp4",
         "format": "mxfp4", "output": "bfloat16", "bias": True},
        # A prefill chunk with 4-bit activations.
        {"name": "linear_prefill_mxfp4", "kind": "linear", "rows": 4096, "columns": 4096, "outputs": 14336,
         "input": "bfloat16", "format": "mxfp4", "output": "bfloat16", "bias": False},
        # One token of Llama-3-8B's gated feed-forward, ready for the linear down.
        {"name": "gated_decode_m1", "kind": "gated", "rows": 1, "columns": 4096, "outputs": 14336, "input": "bfloat16",
         "format": "mxfp8", "output": "mxfp8", "act": "silu"},
        # A ragged chunk of TinyLlama-1.1B's, in floats.
        {"name": "gated_m333", "kind": "gated", "rows": 333, "columns": 2048, "outputs": 5632, "input": "float32",
         "format": "mxfp8", "output": "float32", "act": "silu"},
        # A prefill chunk of Llama-3-8B's, 8-bit rows in and out: the largest call.
        {"name": "gated_prefill_mxfp8", "kind": "gated", "rows": 4096, "columns": 4096, "outputs": 14336,
         "input": "mxfp8", "format": "mxfp8", "output": "mxfp8", "act": "silu"},
    ]


# --------------------------------------------------------------------- drawing


def _log(rng, low, high, multiple=1):
    """A size between low and high, even over its logarithm, as a multiple of `multiple`."""
    value = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(low, min(high, int(round(value / multiple)) * multiple))


def _shape(rng):
    """(columns, outputs) of a linear of the listed models, or in between."""
    if rng.random() < 0.5:
        hidden, inner = rng.choice(((2048, 5632), (4096, 11008), (4096, 14336)))
        return (hidden, inner) if rng.random() < 0.5 else (inner, hidden)
    return _log(rng, 64, 14336, BLOCK), _log(rng, 32, 16384)


def draw(rng):
    while True:
        kind = rng.choice(("norm", "norm", "quantize", "linear", "linear", "linear", "gated", "gated"))
        floats = rng.choice(("float32", "bfloat16", "bfloat16", "float16"))
        rows = 1 if rng.random() < 0.2 else _log(rng, 2, 8192)
        if kind == "norm":
            output = rng.choice((floats, "int8", "q8_0", "mxfp8", "mxfp8", "mxfp4"))
            width = rng.choice((2048, 4096, 5632, 11008, 14336, _log(rng, 64, 16384, BLOCK)))
            if output == floats and rng.random() < 0.3:
                width = _log(rng, 33, 8192)  # no multiple of anything
            case = {"kind": kind, "tokens": rows, "width": width, "input": floats,
                    "residual": rng.choice(("none", floats, "float32")), "output": output}
        elif kind == "quantize":
            case = {"kind": kind, "rows": rows, "columns": _log(rng, 64, 16384, BLOCK), "input": floats,
                    "format": rng.choice(("mxfp4", "mxfp8")), "output": rng.choice((floats, "float32"))}
        else:
            columns, outputs = _shape(rng)
            mx = rng.choice(("mxfp8", "mxfp8", "mxfp4"))
            case = {"kind": kind, "rows": rows, "columns": columns, "outputs": outputs,
                    "input": mx if rng.random() < 0.3 else floats, "format": mx, "output": floats}
            if kind == "linear":
                case["bias"] = rng.random() < 0.5
            else:
                case["act"] = rng.choice(("silu", "silu", "gelu"))
                if rng.random() < 0.5:
                    case["outputs"] = max(BLOCK, outputs // BLOCK * BLOCK)
                    case["output"] = "mxfp8"
        cost = work(case)
        if cost["flops"] <= MOST_FLOPS and cost["bytes"] <= MOST_BYTES:
            return case


# ----------------------------------------------------------------------- costs


def work(case):
    if case["kind"] == "norm":
        size = case["tokens"] * case["width"]
        each = _SIZE[case["input"]] + _SIZE[case["output"]]
        if case["residual"] != "none":
            each += 2 * _SIZE[case["residual"]]
        return {"bytes": int(size * each) + case["width"] * 4, "flops": 5 * size}
    if case["kind"] == "quantize":
        size = case["rows"] * case["columns"]
        each = _SIZE[case["input"]] + 2 * _SIZE[case["format"]] + _SIZE[case["output"]]
        return {"bytes": int(size * each), "flops": 3 * size}
    m, k, n = case["rows"], case["columns"], case["outputs"]
    weights = 2 if case["kind"] == "gated" else 1
    return {"bytes": int(m * k * _SIZE[case["input"]] + weights * n * k * _SIZE["mxfp4"] + m * n * _SIZE[case["output"]]),
            "flops": weights * 2 * m * n * k}


# -------------------------------------------------------------- plain formats

_FP4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _plain_blocks(x, fmt):
    """fp32 rows -> (element values [rows, blocks, 32], exponents [rows, blocks, 1]): a block is 2^exponent times them.

    The exponent is floor(log2) of the block's largest magnitude less that of the format's largest value, at least -127;
    elements are rounded to the nearest, ties to even, and cut to the format's largest.
    """
    top, most, bits, least = (2, 6.0, 1, 0) if fmt == "mxfp4" else (8, 448.0, 3, -6)
    blocks = x.unflatten(-1, (-1, BLOCK))
    amax = blocks.abs().amax(dim=-1, keepdim=True)
    exponent = torch.where(amax > 0, torch.frexp(amax).exponent - 1 - top, -127).clamp(-127, 127)
    blocks = torch.ldexp(torch.ldexp(blocks, -(exponent // 2)), exponent // 2 - exponent)  # 2^127 twice would pass fp32
    step = torch.ldexp(torch.ones_like(blocks), (torch.frexp(blocks).exponent - 1).clamp(min=least) - bits)
    return (torch.round(blocks / step) * step).clamp(-most, most), exponent


def _plain_values(x, fmt):
    """What quantised rows stand for, in fp32."""
    values, exponent = _plain_blocks(x, fmt)
    return torch.ldexp(torch.ldexp(values, exponent // 2), exponent - exponent // 2).flatten(-2)


def _plain_mxfp8(x):
    """(8-bit elements, scales) as torch's types of them."""
    values, exponent = _plain_blocks(x, "mxfp8")
    return values.flatten(-2).to(torch.float8_e4m3fn), (exponent[..., 0] + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _plain_read(values, scales, fmt):
    """Stored blocks -> fp32 rows."""
    scale = torch.ldexp(torch.ones((), device="cuda"), scales.int() - 127)[..., None]
    if fmt == "mxfp8":
        return (values.float().unflatten(-1, (-1, BLOCK)) * scale).flatten(-2)
    codes = torch.stack((values & 15, values >> 4), dim=-1).flatten(-2)
    table = torch.tensor(_FP4 + tuple(-v for v in _FP4), device="cuda")
    return (table[codes.int()].unflatten(-1, (-1, BLOCK)) * scale).flatten(-2)


# -------------------------------------------------------------------- inputs


def _store(x, fmt):
    """Rows in a format's stored form: (values, scales)."""
    values, exponent = _plain_blocks(x, fmt)
    scales = (exponent[..., 0] + 127).to(torch.uint8)
    values = values.flatten(-2)
    if fmt == "mxfp8":
        return values.to(torch.float8_e4m3fn), scales
    code = torch.bucketize(values.abs(), torch.tensor(_FP4, device="cuda")).to(torch.uint8) + 8 * (values < 0).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scales


def _activations(gen, rows, columns):
    """fp32 rows with a few channels of 20 times the others' size, as decoder activations have them."""
    x = torch.randn((rows, columns), generator=gen, device="cuda")
    loud = torch.rand((columns,), generator=gen, device="cuda") < 0.001
    return x * torch.where(loud, 20.0, 1.0)


def _weight(gen, outputs, columns):
    return _store(torch.randn((outputs, columns), generator=gen, device="cuda") * columns**-0.5, "mxfp4")


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    state = dict(case)
    if case["kind"] == "norm":
        state["x"] = torch.randn((case["tokens"], case["width"]), generator=gen, device="cuda").to(_TYPES[case["input"]])
        state["weight"] = 1.0 + 0.2 * torch.randn((case["width"],), generator=gen, device="cuda")
        stream = None
        if case["residual"] != "none":
            stream = (_activations(gen, case["tokens"], case["width"]) * 3.0).to(_TYPES[case["residual"]])
        state["stream"] = stream
        return state
    if case["kind"] == "quantize":
        state["x"] = _activations(gen, case["rows"], case["columns"]).to(_TYPES[case["input"]])
        return state
    x = _activations(gen, case["rows"], case["columns"])
    state["x"] = x.to(_TYPES[case["input"]]) if case["input"] in _TYPES else _store(x, case["input"])
    state["weight"] = _weight(gen, case["outputs"], case["columns"])
    if case["kind"] == "gated":
        state["up"] = _weight(gen, case["outputs"], case["columns"])
    else:
        state["bias"] = torch.randn((case["outputs"],), generator=gen, device="cuda") * 0.1 if case["bias"] else None
    return state


# ---------------------------------------------------------------- plain torch


def _plain_norm(state):
    x, stream, output = state["x"].float(), state["stream"], state["output"]
    added = ()
    if stream is not None:
        added = ((x + stream.float()).to(stream.dtype),)  # the norm is of the stored sum
        x = added[0].float()
    wide = x.double()
    factor = torch.rsqrt((wide * wide).mean(dim=-1, keepdim=True) + EPSILON).float()
    y = x * factor * state["weight"]
    if output in _TYPES:
        return (y.to(_TYPES[output]), *added)
    if output == "mxfp8":
        return (*_plain_mxfp8(y), *added)
    if output == "mxfp4":
        return (_plain_values(y, "mxfp4"), *added)
    if output == "int8":  # one scale a row, of at least 1/127
        amax = y.abs().amax(dim=-1, keepdim=True)
        scale = (amax / torch.full_like(amax, 127.0)).clamp(min=1.0 / 127.0)  # (a number's reciprocal would be multiplied)
        return (torch.round(y / scale).clamp(-127, 127) * scale, *added)
    blocks = y.unflatten(-1, (-1, BLOCK))  # Q8_0: fp16 scales, codes by the reciprocal of the scale before its rounding
    amax = blocks.abs().amax(dim=-1, keepdim=True)
    scale = amax / torch.full_like(amax, 127.0)
    codes = torch.round(blocks * torch.where(scale > 0, 1.0 / scale, 0.0)).clamp(-127, 127)
    return ((codes * scale.half().float()).flatten(-2), *added)


def _plain_activations(state):
    x, fmt = state["x"], state["format"]
    return _plain_values(x.float(), fmt) if state["input"] in _TYPES else _plain_read(*x, fmt)


def _plain_linear(state):
    y = _plain_activations(state) @ _plain_read(*state["weight"], "mxfp4").t()
    if state["bias"] is not None:
        y = y + state["bias"]
    return y.to(_TYPES[state["output"]])


def _plain_gated(state):
    x = _plain_activations(state)
    gate = x @ _plain_read(*state["weight"], "mxfp4").t()
    up = x @ _plain_read(*state["up"], "mxfp4").t()
    if state["act"] == "silu":
        h = gate / (1.0 + torch.exp(-gate)) * up
    else:
        h = 0.5 * gate * (1.0 + torch.erf(gate * math.sqrt(0.5))) * up
    return _plain_mxfp8(h) if state["output"] == "mxfp8" else h.to(_TYPES[state["output"]])


# ------------------------------------------------------------------------ run


def _own_norm(kernels, state):
    output, stream = state["output"], state["stream"]
    args = {"epsilon": EPSILON}
    if output in _TYPES:
        y, added = kernels.add_rms_norm(state["x"], state["weight"], stream, **args)
        return y, added
    if output == "q8_0":
        blocks, added = kernels.add_rms_norm_q8_0(state["x"], state["weight"], stream, **args)
        scale = blocks[..., :2].contiguous().view(torch.float16).float()
        return (blocks[..., 2:].view(torch.int8).float() * scale).flatten(-2), added
    call = {"int8": kernels.add_rms_norm_int8, "mxfp8": kernels.add_rms_norm_mxfp8, "mxfp4": kernels.add_rms_norm_mxfp4}
    values, scales, added = call[output](state["x"], state["weight"], stream, **args)
    if output == "int8":
        return torch.mul(values, scales[:, None]), added
    if output == "mxfp4":
        return kernels.dequantize_mxfp4(values, scales), added
    return values, scales.view(torch.float8_e8m0fnu), added


def _run_own(state):
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from qpu_xla_amd import kernels

    kind, x = state["kind"], state["x"]
    if kind == "norm":
        return _own_norm(kernels, state)
    if kind == "quantize":
        dtype = _TYPES[state["output"]]
        if state["format"] == "mxfp8":
            return kernels.dequantize_mxfp8(*kernels.quantize_mxfp8(x), dtype=dtype)
        return kernels.dequantize_mxfp4(*kernels.quantize_mxfp4(x), dtype=dtype)
    floats = state["input"] in _TYPES
    if kind == "linear":
        dtype = _TYPES[state["output"]]
        if floats:
            return kernels.mxfp4_linear(x, *state["weight"], state["bias"], activations=state["format"], dtype=dtype)
        return kernels.mxfp4_gemm(*x, *state["weight"], state["bias"], dtype=dtype)
    output = "mxfp8" if state["output"] == "mxfp8" else _TYPES[state["output"]]
    if floats:
        h = kernels.mxfp4_gated_linear(x, *state["weight"], *state["up"], activations=state["format"], gate=state["act"],
                                       output=output)
    else:
        h = kernels.mxfp4_gated_gemm(*x, *state["weight"], *state["up"], gate=state["act"], output=output)
    return (h[0], h[1].view(torch.float8_e8m0fnu)) if output == "mxfp8" else h


def run(state):
    if own:
        return _run_own(state)
    kind = state["kind"]
    if kind == "norm":
        return _plain_norm(state)
    if kind == "quantize":
        return _plain_values(state["x"].float(), state["format"]).to(_TYPES[state["output"]])
    return _plain_linear(state) if kind == "linear" else _plain_gated(state)


# ---------------------------------------------------------------------- exact


def _grid(fmt):
    """The format's magnitudes in order, from its bits."""
    if fmt == "mxfp4":
        codes, exponent_bits, mantissa_bits, bias = torch.arange(8), 2, 1, 1
    else:
        codes, exponent_bits, mantissa_bits, bias = torch.arange(127), 4, 3, 7  # code 127 is no number
    exponent, mantissa = codes >> mantissa_bits, (codes & ((1 << mantissa_bits) - 1)).double() / (1 << mantissa_bits)
    assert int(exponent.max()) < 1 << exponent_bits
    return torch.where(exponent > 0, (1 + mantissa) * 2.0 ** (exponent - bias), mantissa * 2.0 ** (1 - bias)).cuda()


def _exact_blocks(x, fmt):
    """64-bit rows -> (elements, scales) by searching the format's values; equal distances go to the even code."""
    grid = _grid(fmt)
    blocks = x.reshape(*x.shape[:-1], -1, BLOCK)
    amax = blocks.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.floor(torch.log2(amax.clamp(min=2.0**-140))) - torch.floor(torch.log2(grid[-1])))
    scale = scale.clamp(min=2.0**-127)
    borders = (grid[1:] + grid[:-1]) / 2
    size = (blocks / scale).abs()
    below, above = torch.bucketize(size, borders), torch.bucketize(size, borders, right=True)
    index = torch.where(below % 2 == 0, below, above)
    return torch.copysign(grid[index], blocks), scale


def _exact_values(x, fmt):
    elements, scale = _exact_blocks(x, fmt)
    return (elements * scale).flatten(-2)


def _exact_mxfp8(x):
    elements, scale = _exact_blocks(x, "mxfp8")
    return elements.flatten(-2), scale[..., 0]


def _exact_read(values, scales, fmt):
    if fmt == "mxfp8":
        elements = values.double()
    else:
        grid = _grid("mxfp4")
        pair = torch.stack((values % 16, values // 16), -1).long().flatten(-2)
        elements = grid[pair % 8] * (1 - 2 * (pair // 8))
    return elements * (2.0 ** (scales.double() - 127)).repeat_interleave(BLOCK, -1)


def _exact_norm(state):
    x, stream, output = state["x"].double(), state["stream"], state["output"]
    added = ()
    if stream is not None:
        total = x + stream.double()
        added = (total,)
        x = total.float().to(stream.dtype).double()  # what the norm is defined on
    factor = 1.0 / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPSILON)
    if output in _TYPES:
        return (x * factor * state["weight"].double(), *added)
    # Codes are defined on the row after the roundings to 32 bits: of the factor and of both products.
    y = ((x * factor.float().double()).float().double() * state["weight"].double()).float().double()
    if output == "mxfp8":
        return (*_exact_mxfp8(y), *added)
    if output == "mxfp4":
        return (_exact_values(y, "mxfp4"), *added)
    if output == "int8":
        scale = (y.abs().amax(-1, keepdim=True) / 127).float().double().clamp(min=float(torch.tensor(1 / 127)))
        return (torch.round((y / scale).float()).double() * scale, *added)
    blocks = y.reshape(*y.shape[:-1], -1, BLOCK)
    scale = (blocks.abs().amax(-1, keepdim=True) / 127).float().double()
    inverse = torch.where(scale > 0, (1 / scale).float().double(), 0.0)
    return ((torch.round((blocks * inverse).float()).double() * scale.half().double()).flatten(-2), *added)


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "norm":
        return _exact_norm(state)
    fmt = case["format"]
    if case["kind"] == "quantize":
        return _exact_values(state["x"].double(), fmt)
    x = _exact_values(state["x"].double(), fmt) if case["input"] in _TYPES else _exact_read(*state["x"], fmt)
    gate = torch.nn.functional.linear(x, _exact_read(*state["weight"], "mxfp4"))
    if case["kind"] == "linear":
        return gate if state["bias"] is None else gate + state["bias"].double()
    up = torch.nn.functional.linear(x, _exact_read(*state["up"], "mxfp4"))
    if case["act"] == "silu":
        h = gate * torch.sigmoid(gate) * up
    else:
        h = gate * 0.5 * torch.erfc(-gate / math.sqrt(2.0)) * up
    return _exact_mxfp8(h) if case["output"] == "mxfp8" else h
