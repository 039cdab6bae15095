"""Microscaled rows in plain 64-bit arithmetic on the CPU: what the kernels are compared with."""

import math

import torch

BLOCK = 32


def numbers(bits: int) -> torch.Tensor:
    """The format's numbers that are not negative, by code."""
    if bits == 4:
        return torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
    return torch.tensor([(code % 8) * 2.0**-9 if code < 8 else (1 + code % 8 / 8) * 2.0 ** (code // 8 - 7) for code in range(127)], dtype=torch.float64)


def powers() -> torch.Tensor:
    return torch.tensor([2.0 ** (byte - 127) for byte in range(255)] + [math.nan], dtype=torch.float64)


def padded(width: int) -> int:
    return -(-width // 128) * 128


def quantise(values: torch.Tensor, bits: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes ``[rows, padded]`` (one per element) and scale bytes ``[rows, padded / 32]`` of rows of finite numbers, or blocks with others."""
    rows, width = values.shape
    blocks = torch.zeros(rows, padded(width), dtype=torch.float64)
    blocks[:, :width] = values.double()
    blocks = blocks.view(rows, -1, BLOCK)
    finite = torch.isfinite(blocks).all(dim=-1)
    blocks = torch.where(finite[..., None], blocks, 0.0)
    exponent = torch.frexp(blocks.abs().amax(dim=-1)).exponent - 1 - (8 if bits == 8 else 2)
    byte = torch.where(blocks.abs().amax(dim=-1) > 0, exponent + 127, 0).clamp(min=0)
    sizes = (blocks / powers()[byte][..., None]).abs()
    grid = numbers(bits)
    upper = torch.bucketize(sizes, grid).clamp(max=len(grid) - 1)  # the first number that is not smaller
    lower = (upper - 1).clamp(min=0)
    to_lower, to_upper = sizes - grid[lower], grid[upper] - sizes
    code = torch.where((to_upper < to_lower) | ((to_upper == to_lower) & (upper % 2 == 0)) | (to_upper <= 0), upper, lower)
    code = code + (len(grid) + 1 if bits == 8 else len(grid)) * torch.signbit(blocks)
    return torch.where(finite[..., None], code, 0).view(rows, -1), torch.where(finite, byte, 255)


def stands_for(codes: torch.Tensor, scale_bytes: torch.Tensor, bits: int) -> torch.Tensor:
    """The values, ``[rows, padded]`` in 64 bits."""
    half = 128 if bits == 8 else 8
    grid = torch.cat([numbers(bits), torch.tensor([math.nan] * (half - len(numbers(bits))), dtype=torch.float64)])
    elements = torch.where(codes >= half, -grid[codes % half], grid[codes % half])
    return (elements.view(codes.shape[0], -1, BLOCK) * powers()[scale_bytes.long()][..., None]).view(codes.shape[0], -1)


def pack(codes: torch.Tensor, scale_bytes: torch.Tensor, bits: int, rest: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """The two tensors of bytes that the kernels take; ``rest`` in the scales of rows that do not exist."""
    rows, columns = codes.shape
    packed = codes if bits == 8 else codes[:, 0::2] + 16 * codes[:, 1::2]
    scales = torch.full((-(-rows // 128), columns // 128, 512), rest, dtype=torch.uint8)
    row, block = torch.arange(rows)[:, None], torch.arange(columns // BLOCK)[None, :]
    scales[row // 128, block // 4, row % 32 * 16 + row % 128 // 32 * 4 + block % 4] = scale_bytes.to(torch.uint8)
    return packed.to(torch.uint8).contiguous(), scales


def unpack(packed: torch.Tensor, scales: torch.Tensor, bits: int) -> tuple[torch.Tensor, torch.Tensor]:
    """The reverse of :func:`pack`."""
    rows = packed.shape[0]
    codes = packed.long() if bits == 8 else torch.stack([packed.long() & 15, packed.long() >> 4], dim=-1).view(rows, -1)
    row, block = torch.arange(rows)[:, None], torch.arange(codes.shape[1] // BLOCK)[None, :]
    return codes, scales.long()[row // 128, block // 4, row % 32 * 16 + row % 128 // 32 * 4 + block % 4]


def through(values: torch.Tensor, bits: int) -> torch.Tensor:
    """What rows become in microscaled form, in 64 bits."""
    return stands_for(*quantise(values, bits), bits)[:, : values.shape[1]]


def activate(gate: torch.Tensor, up: torch.Tensor, activation: str, limit: float = 0.0) -> torch.Tensor:
    if activation == "silu":
        return up * gate * torch.sigmoid(gate)
    if activation == "gelu":
        return up * 0.5 * gate * (1 + torch.erf(gate / math.sqrt(2.0)))
    if activation == "sigmoid_limit":
        g = gate.clamp(max=limit)
        return g * torch.sigmoid(1.702 * g) * (up.clamp(-limit, limit) + 1)
    return up * gate
