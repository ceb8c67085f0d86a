"""Operators on matrices in microscaled 4-bit floating point, as cases that can be timed and compared.

A matrix in this form is cut, along its rows, into blocks of 32 entries.  A block has a scale, a power of
two held in a byte, and its entries are 4-bit floats (sign, two bits of exponent, one of mantissa):

* ``quantize``: ``rows`` x ``columns`` numbers to this form and back to the values that it stands for;
* ``linear``: ``x W^T`` with a quantised weight ``[outputs, columns]`` under rows of ``dtype`` as they are (what a
  model with 4-bit weights computes for a step's tokens);
* ``quantized_linear``: the same with the rows quantised first (4-bit weights and activations).
"""

from __future__ import annotations

import math

import torch

own = False      # True: the calls that a user of the framework makes; False: elementary operations

DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
BLOCK = 32
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
MAX_FLOPS = 2 * 8192 * 4096 * 24576     # of a drawn case: the largest listed one's
MAX_CELLS = 2048 * 9728                 # of a drawn quantisation


def listed():
    return [
        # one token's hidden row, ahead of a product with quantised activations
        {"name": "quantize_token", "kind": "quantize", "rows": 1, "columns": 2560, "dtype": "bfloat16"},
        # a small matrix whose rows end inside a block
        {"name": "quantize_odd", "kind": "quantize", "rows": 37, "columns": 1000, "dtype": "float32"},
        # what a prompt of 2,048 tokens brings to the down projection of a 4B model
        {"name": "quantize_prompt", "kind": "quantize", "rows": 2048, "columns": 9728, "dtype": "bfloat16"},
        # one user's next token: the q, k and v projection of a 4B model
        {"name": "linear_token", "kind": "linear", "rows": 1, "columns": 2560, "outputs": 6144, "dtype": "bfloat16", "bias": False},
        # eight users' next tokens: the down projection
        {"name": "linear_batch_8", "kind": "linear", "rows": 8, "columns": 9728, "outputs": 2560, "dtype": "bfloat16", "bias": False},
        # a batch of thirty-two: gate and up projection of a 14B model
        {"name": "linear_batch_32", "kind": "linear", "rows": 32, "columns": 5120, "outputs": 34816, "dtype": "bfloat16", "bias": False},
        # the 32-bit path on odd sizes, with a bias
        {"name": "linear_odd", "kind": "linear", "rows": 5, "columns": 1000, "outputs": 1333, "dtype": "float32", "bias": True},
        # a prompt of 2,048 tokens: gate and up projection of an 8B model
        {"name": "linear_prompt", "kind": "linear", "rows": 2048, "columns": 4096, "outputs": 24576, "dtype": "bfloat16", "bias": False},
        # three users' next tokens with quantised activations: the output projection of an 8B model
        {"name": "quantized_linear_batch_3", "kind": "quantized_linear", "rows": 3, "columns": 4096, "outputs": 4096, "dtype": "bfloat16",
         "bias": False},
        # a short prompt of an odd length, sizes that fill no tile, a bias
        {"name": "quantized_linear_odd", "kind": "quantized_linear", "rows": 77, "columns": 1096, "outputs": 515, "dtype": "float32",
         "bias": True},
        # prompts of 8,192 tokens in all: gate and up projection of an 8B model
        {"name": "quantized_linear_prompt", "kind": "quantized_linear", "rows": 8192, "columns": 4096, "outputs": 24576,
         "dtype": "bfloat16", "bias": False},
    ]


def _between(rng, low, high):
    """A whole number, spread evenly over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    kind = rng.choice(["quantize", "linear", "linear", "quantized_linear"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    # widths are multiples of 8 in earnest, now and then any number
    columns = _between(rng, 32, 12288)
    if rng.random() < 0.7:
        columns = (columns + 7) // 8 * 8
    if kind == "quantize":
        rows = _between(rng, 1, max(1, min(8192, MAX_CELLS // columns)))
        return {"kind": kind, "rows": rows, "columns": columns, "dtype": dtype}
    outputs = _between(rng, 8, 24576)
    rows = _between(rng, 1, 4096)
    if dtype == "float32":      # the 32-bit path is for checking results: small batches
        rows = min(rows, 512)
    rows = max(1, min(rows, MAX_FLOPS // (2 * columns * outputs)))
    return {"kind": kind, "rows": rows, "columns": columns, "outputs": outputs, "dtype": dtype, "bias": rng.random() < 0.25}


# ------------------------------------------------------------------ inputs


def _activations(case, g):
    """Rows as a norm with gains leaves them: most entries near one, a few channels far larger."""
    rows, columns = case["rows"], case["columns"]
    gain = 0.5 + torch.rand(columns, generator=g, device="cuda")
    loud = torch.rand(columns, generator=g, device="cuda") < 0.01
    gain = torch.where(loud, gain * 12.0, gain)
    x = torch.randn((rows, columns), generator=g, device="cuda") * gain
    return x.to(DTYPES[case["dtype"]])


def _weight(case, g):
    """A projection's weight: normal, each output with a spread of its own."""
    n, k = case["outputs"], case["columns"]
    spread = 0.02 * (0.5 + torch.rand((n, 1), generator=g, device="cuda"))
    return torch.randn((n, k), generator=g, device="cuda").mul_(spread)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    made = {"x": _activations(case, g), "codes": None, "scales": None, "bias": None}
    if case["kind"] != "quantize":
        # the stored form: two codes a byte, the first in the low half, and a scale byte per block
        codes, exponents = _quantize(_weight(case, g))
        codes = codes.reshape(codes.shape[0], -1)[:, :case["columns"]]
        if case["columns"] % 2:
            codes = torch.nn.functional.pad(codes, (0, 1))
        made["codes"] = (codes[:, 0::2] | codes[:, 1::2] << 4).contiguous()
        made["scales"] = (exponents + 127).to(torch.uint8)
        if case["bias"]:
            made["bias"] = torch.randn(case["outputs"], generator=g, device="cuda").to(DTYPES[case["dtype"]])
    return made


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if own:
        from thing_htn_2026_b200 import ops
        state["ops"] = ops
        state["err"] = ops.new_error_word("cuda")
        if case["kind"] != "quantize":
            state["weight"] = ops.mx4_from_parts(state.pop("codes"), state.pop("scales"), case["columns"])
    return state


# ------------------------------------------------------------------ the plain forms


def _blocks(x):
    """Rows cut into blocks, the last filled up with zeros: [rows, blocks, 32] float32."""
    rows, columns = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -columns % BLOCK))
    return x.reshape(rows, -1, BLOCK)


def _quantize(x):
    """(codes [rows, blocks, 32] uint8, scale exponents [rows, blocks] int32) of finite numbers."""
    v = _blocks(x)
    top = v.abs().amax(dim=-1)
    _, e = torch.frexp(top)                                    # top = m 2^e with 1/2 <= m < 1
    exponents = torch.where(top > 0, e - 1 - 2, -127).clamp(-127, 127).to(torch.int32)
    # (two steps: 2^127 alone is a float32, 2^128 is not)
    half = torch.div(-exponents, 2, rounding_mode="floor")
    scaled = torch.ldexp(torch.ldexp(v, half[..., None]), (-exponents - half)[..., None])
    size = scaled.abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    size = (torch.round(size / step) * step).clamp(max=6.0)    # (round: ties to even)
    # the code of a magnitude: twice the number below 2, then 5, 6 and 7 for 3, 4 and 6
    code = torch.where(size <= 2, size * 2, torch.where(size <= 4, size + 2, size + 1))
    return code.to(torch.uint8) | (torch.signbit(v).to(torch.uint8) << 3), exponents


def _values(codes, exponents, columns):
    """The float32 numbers [rows, columns] that codes and exponents stand for."""
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=codes.device)
    v = torch.ldexp(table[codes.int()], exponents[..., None])
    return v.reshape(v.shape[0], -1)[:, :columns]


def _stored_values(codes, scales, columns):
    """The same from the stored form."""
    pairs = torch.stack((codes & 15, codes >> 4), dim=-1).reshape(codes.shape[0], -1)
    pairs = torch.nn.functional.pad(pairs, (0, scales.shape[1] * BLOCK - pairs.shape[1]))
    return _values(pairs.reshape(codes.shape[0], -1, BLOCK), scales.to(torch.int32) - 127, columns)


def run(state):
    case = state["case"]
    if own:
        ops, x = state["ops"], state["x"]
        if case["kind"] == "quantize":
            return ops.dequantize_mx4(ops.quantize_mx4(x), x.dtype)
        rows = ops.quantize_mx4(x) if case["kind"] == "quantized_linear" else x
        return ops.linear_mx4(rows, state["weight"], out_dtype=x.dtype, bias=state["bias"], err=state["err"])
    x = state["x"]
    if case["kind"] == "quantize":
        return _values(*_quantize(x), case["columns"]).to(x.dtype)
    w = _stored_values(state["codes"], state["scales"], case["columns"])
    rows = _values(*_quantize(x), case["columns"]) if case["kind"] == "quantized_linear" else x.float()
    y = rows @ w.t()
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(x.dtype)


def work(case):
    rows, columns = case["rows"], case["columns"]
    size = 2 if case["dtype"] == "bfloat16" else 4
    blocks = -(-columns // BLOCK)
    held = (columns + 1) // 2 + blocks                         # bytes of a row in 4 bits
    if case["kind"] == "quantize":
        # the numbers in, codes and scales out; codes and scales in, their values out
        return {"bytes": rows * (2 * size * columns + 2 * held), "flops": 2 * rows * columns}
    n = case["outputs"]
    moved = rows * columns * size + n * held + rows * n * size + (n * size if case["bias"] else 0)
    return {"bytes": moved, "flops": 2 * rows * columns * n}


# ------------------------------------------------------------------ from the definition, in 64 bits


def _nearest(v):
    """The nearest representable number of each entry of v (float64, scaled), by its place among the midpoints; of two
    equally near ones that with the even code."""
    table = torch.tensor(MAGNITUDES, dtype=torch.float64, device=v.device)
    middle = (table[1:] + table[:-1]) / 2
    size = v.abs().contiguous()
    code = torch.bucketize(size, middle)                       # how many midpoints lie below
    tie = (size == middle[code.clamp(max=6)]) & (code % 2 == 1) & (code < 7)
    return torch.copysign(table[code + tie.long()], v)


def _quantized_values(x):
    """What the quantised rows stand for, in float64."""
    out = []
    for piece in torch.split(x, 512):
        v = _blocks(piece).double()
        top = v.abs().amax(dim=-1, keepdim=True)
        # the largest power of two that is not above the block's largest entry
        power = torch.exp2(torch.floor(torch.log2(top)))
        power = torch.where(power > top, power / 2, torch.where(power * 2 <= top, power * 2, power))
        scale = torch.where(top > 0, power / 4, 1.0).clamp(2.0 ** -127, 2.0 ** 127)
        out.append((_nearest(v / scale) * scale).flatten(1)[:, :x.shape[1]])
    return torch.cat(out)


def exact(case, seed):
    made = _inputs(case, seed)
    if case["kind"] == "quantize":
        return _quantized_values(made["x"])
    low, high = (made["codes"] & 15).long(), (made["codes"] >> 4).long()
    codes = torch.stack((low, high), dim=-1).flatten(1)[:, :case["columns"]]
    table = torch.tensor(MAGNITUDES, dtype=torch.float64, device=codes.device)
    w = table[codes & 7]
    w = torch.where(codes >= 8, -w, w)
    w *= torch.exp2(made["scales"].double() - 127).repeat_interleave(BLOCK, dim=1)[:, :case["columns"]]
    rows = _quantized_values(made["x"]) if case["kind"] == "quantized_linear" else made["x"].double()
    y = rows @ w.t()
    return y if made["bias"] is None else y + made["bias"].double()
