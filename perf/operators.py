"""Microscaled operators, as cases that can be timed and compared: rows of numbers held in 8 or 4 bits with a power of two as the scale of
every 32 of them (the formats of the OCP microscaling specification: e4m3 or e2m1 elements, e8m0 scales), and what a feed-forward in them needs:

* ``quantise``  rows of bfloat16 or float32 into 8 or 4 bits, and the values that these stand for;
* ``norm``      a sublayer's output added to the 32-bit residual stream, and the RMS norm of the sum in 8 (or 4) bits;
* ``linear``    the product of such rows, in 8 or 4 bits, with a weight in 4 bits;
* ``gated``     ``up(x) * silu(gate(x))`` of such rows and two weights in 4 bits, in 8 bits again (the next product's rows).

Sizes are those of the random-weight presets (width 1024 and feed-forwards of 4,608, 1536 and 6,912, 2048 and 8,192), from a single decoded
token to long prompts, and odd ones.

Rows in microscaled form are two tensors of bytes.  ``codes [rows, padded * bits / 8]``: the elements, ``padded`` columns of them (the width
made up to a multiple of 128 with zeros), of 4-bit elements the even column in the lower half of its byte.  ``scales [row tiles, padded / 128,
512]``: a byte ``b`` stands for ``2^(b - 127)`` (255: not a number); that of row ``r`` and columns ``32 c`` to ``32 c + 31`` is byte
``(r % 32) * 16 + (r % 128) // 32 * 4 + c % 4`` of the tile ``[r // 128, c // 4]``.
"""

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
BLOCK = 32  # elements under one scale
EPS = 1e-5
LARGEST_EXPONENT = {8: 8, 4: 2}  # of the largest element: 448 = 1.75 * 2^8, 6 = 1.5 * 2^2

# ------------------------------------------------------------------------------------------------------------------ cases


def _quantise(name, tokens, width, bits, dtype):
    return {"name": name, "kind": "quantise", "tokens": tokens, "width": width, "bits": bits, "dtype": dtype}


def _norm(name, tokens, width, bits, dtype):
    return {"name": name, "kind": "norm", "tokens": tokens, "width": width, "bits": bits, "dtype": dtype}


def _linear(name, tokens, width, rows, bits, dtype):
    return {"name": name, "kind": "linear", "tokens": tokens, "width": width, "rows": rows, "bits": bits, "dtype": dtype}


def _gated(name, tokens, width, rows, bits):
    return {"name": name, "kind": "gated", "tokens": tokens, "width": width, "rows": rows, "bits": bits, "dtype": "bfloat16"}


def listed():
    return [
        # the rows of eight users' next tokens, between an attention layer and its output projection
        _quantise("quantise_8_rows", 8, 2048, 8, "bfloat16"),
        # a feed-forward's weight brought into 4 bits when a model is loaded
        _quantise("quantise_weight_4_bits", 8192, 2048, 4, "bfloat16"),
        # an odd width: the last block is a part of one
        _quantise("quantise_float32_777x1001", 777, 1001, 4, "float32"),
        # one user's next token: the smallest call
        _norm("norm_1_token", 1, 2048, 8, "bfloat16"),
        # a prompt at the 1.2B width
        _norm("norm_prompt_4096", 4096, 2048, 8, "bfloat16"),
        # one user's next token through a feed-forward's second product
        _linear("linear_1_token", 1, 8192, 2048, 8, "bfloat16"),
        # eight users' next tokens through a square projection, into 32 bits
        _linear("linear_8_tokens", 8, 2048, 2048, 8, "float32"),
        # an odd number of tokens, odd width and rows
        _linear("linear_333_odd", 333, 1001, 777, 4, "bfloat16"),
        # a long prompt through a feed-forward's second product, rows in 8 bits and in 4
        _linear("linear_prompt_4096_8_bits", 4096, 8192, 2048, 8, "bfloat16"),
        _linear("linear_prompt_4096_4_bits", 4096, 8192, 2048, 4, "bfloat16"),
        # eight users' next tokens through a feed-forward's first two products
        _gated("gated_8_tokens", 8, 2048, 8192, 8),
        # a prompt of 777 tokens through the 700M shape's
        _gated("gated_prompt_777", 777, 1536, 6912, 8),
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["quantise", "norm", "linear", "linear", "gated"])
    bits = rng.choice([8, 8, 4])
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    if kind in ("quantise", "norm"):
        return {"kind": kind, "tokens": _spread(rng, 1, 8192), "width": _spread(rng, 1, 8192) if kind == "quantise" else _spread(rng, 32, 8192), "bits": bits, "dtype": dtype}
    while True:
        tokens, width, rows = _spread(rng, 1, 8192), _spread(rng, 32, 8192), _spread(rng, 16, 16384)
        if tokens * width * rows * (2 if kind == "gated" else 1) <= 4096 * 8192 * 2048:
            break
    return {"kind": kind, "tokens": tokens, "width": width, "rows": rows, "bits": bits, "dtype": dtype if kind == "linear" else "bfloat16"}


# ------------------------------------------------------------------------------------------------------------------ plain forms


def _padded(width):
    return -(-width // 128) * 128


def _power(exponents):
    """``2^exponents`` in float32, from -127 (a subnormal) to 127, exact (which ``pow`` and ``ldexp`` on the GPU are not)."""
    return torch.where(exponents >= -126, (exponents + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _rounded(values, bits):
    """Float32 values, already divided by their scales, to the nearest of the format's, ties to the even code; what is larger than the largest becomes that."""
    if bits == 8:
        return values.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).float()
    size = values.abs()
    step = torch.where(size < 2.0, 0.5, torch.where(size < 4.0, 1.0, 2.0))
    return torch.copysign((torch.round(size / step) * step).clamp(max=6.0), values)


def _blocks(values, bits):
    """Float32 rows in blocks of 32, the last one made up with zeros: the elements ``[rows, blocks, 32]`` and the scales' exponents ``[rows, blocks]``.
    The scale is the power of two that brings the largest value of a block under the next power of two above the largest element's."""
    rows, width = values.shape
    blocks = torch.nn.functional.pad(values, (0, -width % BLOCK)).view(rows, -1, BLOCK)
    largest = blocks.abs().amax(dim=-1)
    exponents = (torch.frexp(largest).exponent - 1 - LARGEST_EXPONENT[bits]).clamp(min=-127)
    exponents = torch.where(largest == 0, -127, exponents)
    return _rounded(blocks * _power(-exponents).unsqueeze(-1), bits), exponents


def _quantised_values(values, bits):
    """What float32 rows become in microscaled form, as float32."""
    rows, width = values.shape
    elements, exponents = _blocks(values, bits)
    return (elements * _power(exponents).unsqueeze(-1)).reshape(rows, -1)[:, :width]


def _microscaled(values, bits):
    """Codes and scales of float32 rows, as bytes."""
    rows, width = values.shape
    padded = _padded(width)
    elements, exponents = _blocks(torch.nn.functional.pad(values, (0, padded - width)), bits)
    elements = elements.view(rows, padded)
    if bits == 8:
        codes = elements.to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=values.device)
        code = torch.bucketize(elements.abs(), grid) + 8 * torch.signbit(elements)
        codes = (code[:, 0::2] + 16 * code[:, 1::2]).to(torch.uint8)
    tiles = torch.zeros(-(-rows // 128) * 128, padded // BLOCK, dtype=torch.uint8, device=values.device)
    tiles[:rows] = (exponents + 127).to(torch.uint8)
    scales = tiles.view(-1, 4, 32, padded // 128, 4).permute(0, 3, 2, 1, 4).reshape(-1, padded // 128, 512)
    return codes.contiguous(), scales.contiguous()


def _values(codes, scales, width, bits):
    """The float32 rows that codes and scales stand for."""
    rows = codes.shape[0]
    if bits == 8:
        elements = codes.view(torch.float8_e4m3fn).float()
    else:
        grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=codes.device)
        elements = grid[torch.stack([codes & 15, codes >> 4], dim=-1).int()].view(rows, -1)
    exponents = scales.view(scales.shape[0], scales.shape[1], 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(scales.shape[0] * 128, -1)[:rows].int() - 127
    return (elements.view(rows, -1, BLOCK) * _power(exponents).unsqueeze(-1)).view(rows, -1)[:, :width]


# ------------------------------------------------------------------------------------------------------------------ what is measured


def _activations(rows, width, generator, dtype=torch.float32):
    """Rows as a model's layers hand them on: some channels much larger than others, and one row in sixteen empty, as rows that pad a batch are."""
    channels = torch.exp(torch.randn(width, generator=generator, device=DEVICE))
    values = torch.randn(rows, width, generator=generator, device=DEVICE) * channels
    values[7::16] = 0.0
    return values.to(dtype)


def prepare(case, seed):
    generator = torch.Generator(device=DEVICE)
    generator.manual_seed(seed)
    tokens, width, bits, dtype = case["tokens"], case["width"], case["bits"], DTYPES[case["dtype"]]
    state = dict(case)
    if case["kind"] == "quantise":
        state["x"] = _activations(tokens, width, generator, dtype)
    elif case["kind"] == "norm":
        state["stream"] = _activations(tokens, width, generator)
        state["delta"] = _activations(tokens, width, generator, dtype)
        state["weight"] = 1.0 + 0.1 * torch.randn(width, generator=generator, device=DEVICE)
    else:
        state["x"] = _microscaled(_activations(tokens, width, generator), bits)
        for name in ("up", "gate") if case["kind"] == "gated" else ("weight",):
            state[name] = _microscaled(torch.randn(case["rows"], width, generator=generator, device=DEVICE) / math.sqrt(width), 4)
    return state


def run(state):
    kind, width, bits, dtype = state["kind"], state["width"], state["bits"], DTYPES[state["dtype"]]
    if own:
        from lalamo_b200 import ops

        if kind == "quantise":
            return ops.microscale(state["x"], bits).values(dtype)
        if kind == "norm":
            stream = torch.empty_like(state["stream"])
            rows = ops.rmsnorm_microscaled(state["stream"], state["weight"], EPS, delta=state["delta"], sum_out=stream, bits=bits)
            return stream, rows.values(torch.bfloat16)
        x = ops.Microscaled(*state["x"], width, bits)
        if kind == "linear":
            return ops.linear_microscaled(x, ops.Microscaled(*state["weight"], width, 4), dtype)
        rows = ops.gated_linear_microscaled(x, ops.Microscaled(*state["up"], width, 4), ops.Microscaled(*state["gate"], width, 4), "silu")
        return rows.values(dtype)
    if kind == "quantise":
        return _quantised_values(state["x"].float(), bits).to(dtype)
    if kind == "norm":
        stream = state["stream"] + state["delta"].float()
        normed = stream * torch.rsqrt(stream.square().mean(dim=-1, keepdim=True) + EPS) * state["weight"]
        return stream, _quantised_values(normed, bits).to(torch.bfloat16)
    x = _values(*state["x"], width, bits)
    if kind == "linear":
        return (x @ _values(*state["weight"], width, 4).t()).to(dtype)
    up, gate = x @ _values(*state["up"], width, 4).t(), x @ _values(*state["gate"], width, 4).t()
    return _quantised_values(up * (gate / (1.0 + torch.exp(-gate))), 8).to(dtype)


def work(case):
    tokens, width, bits = case["tokens"], case["width"], case["bits"]
    size = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "quantise":
        return {"bytes": 2 * tokens * width * size, "flops": 3 * tokens * width}
    if case["kind"] == "norm":
        return {"bytes": tokens * width * (4 + size + 4 + 2) + 4 * width, "flops": 8 * tokens * width}
    rows, weights = case["rows"], 2 if case["kind"] == "gated" else 1
    read = (tokens * bits + weights * rows * 4) * width / 8 + (tokens + weights * rows) * -(-width // BLOCK)
    return {"bytes": read + tokens * rows * size, "flops": 2 * weights * tokens * width * rows}


# ------------------------------------------------------------------------------------------------------------------ in 64 bits


def _format(bits):
    """The numbers of the format that are not negative, in the order of their codes, in 64 bits."""
    mantissa_bits, bias, count = (3, 7, 127) if bits == 8 else (1, 1, 8)  # of e4m3, code 127 is not a number
    numbers = []
    for code in range(count):
        exponent, mantissa = code >> mantissa_bits, code & ((1 << mantissa_bits) - 1)
        one = 1 if exponent else 0
        numbers.append((one + mantissa / (1 << mantissa_bits)) * 2.0 ** (max(exponent, 1) - bias))
    return torch.tensor(numbers, dtype=torch.float64, device=DEVICE)


def _powers():
    """``2^(byte - 127)`` for the bytes 0 to 254, and not a number for 255, in 64 bits."""
    return torch.tensor([2.0 ** (byte - 127) for byte in range(255)] + [math.nan], dtype=torch.float64, device=DEVICE)


def _exactly_quantised(values, bits):
    """Rows in 64 bits to the numbers their microscaled form stands for."""
    numbers = _format(bits)
    middles = (numbers[1:] + numbers[:-1]) / 2
    rows, width = values.shape
    count = -(-width // BLOCK)
    block = torch.arange(width, device=DEVICE) // BLOCK
    largest = torch.zeros(rows, count, dtype=torch.float64, device=DEVICE).scatter_reduce(1, block.expand(rows, width), values.abs(), "amax")
    mantissa, exponent = torch.frexp(largest)
    byte = torch.where(largest > 0, exponent - 1 - int(math.log2(float(numbers[-1]))) + 127, 0).clamp(min=0)
    scale = _powers()[byte][:, block]
    size = (values / scale).abs()
    lower = torch.bucketize(size, middles)  # the first code whose middle to the next is not below
    tie = (size == middles[lower.clamp(max=len(middles) - 1)]) & (lower < len(middles)) & (lower % 2 == 1)
    return torch.sign(values) * numbers[(lower + tie).clamp(max=len(numbers) - 1)] * scale


def _exact_values(codes, scales, width, bits):
    rows = codes.shape[0]
    column = torch.arange(width, device=DEVICE)
    numbers = _format(bits)
    numbers = torch.cat([numbers, numbers.new_full((128 - len(numbers),), math.nan)]) if bits == 8 else numbers
    code = codes[:, column].int() if bits == 8 else (codes[:, column // 2].int() >> (column % 2 * 4)) & 15
    half = 128 if bits == 8 else 8
    elements = numbers[code % half] * (1 - 2 * (code // half))
    row, block = torch.arange(rows, device=DEVICE)[:, None], column // BLOCK
    scale = scales[row // 128, block // 4, row % 32 * 16 + row % 128 // 32 * 4 + block % 4]
    return elements * _powers()[scale.int()]


def exact(case, seed):
    state = prepare(case, seed)
    kind, width, bits = case["kind"], case["width"], case["bits"]
    if kind == "quantise":
        return _exactly_quantised(state["x"].double(), bits)
    if kind == "norm":
        stream = state["stream"].double() + state["delta"].double()
        size = torch.sqrt((stream * stream).sum(dim=-1, keepdim=True) / width + EPS)
        return stream, _exactly_quantised(stream / size * state["weight"].double(), bits)
    x = _exact_values(*state["x"], width, bits)
    if kind == "linear":
        return x @ _exact_values(*state["weight"], width, 4).t()
    up, gate = (x @ _exact_values(*state[name], width, 4).t() for name in ("up", "gate"))
    return _exactly_quantised(up * gate * torch.sigmoid(gate), 8)
