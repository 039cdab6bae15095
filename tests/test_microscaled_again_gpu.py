"""Microscaled operators called again: the same bits as a call by itself, with nothing waited for between calls, other calls before and after, and few and many
CTAs that share a product's K."""

import pytest
import torch

from lalamo_b200 import ops

pytestmark = pytest.mark.gpu
DEVICE = "cuda"


def rows_of(count, width, bits, seed):
    generator = torch.Generator(device=DEVICE).manual_seed(seed)
    return ops.microscale(torch.randn(count, width, generator=generator, device=DEVICE) * torch.exp(torch.randn(width, generator=generator, device=DEVICE)), bits)


def same(one, other):
    if isinstance(one, ops.Microscaled):
        return torch.equal(one.codes, other.codes) and torch.equal(one.values(torch.float32), other.values(torch.float32))
    return torch.equal(one, other)


def check_again(calls, times=20):
    """`calls` one after the other with a wait between them, then in turn without: all of them the same bits."""
    want = []
    for call in calls:
        torch.cuda.synchronize()
        want.append(call())
    torch.cuda.synchronize()
    got = [[call() for call in calls] for _ in range(times)]
    torch.cuda.synchronize()
    for turn, outputs in enumerate(got):
        for place, (output, expected) in enumerate(zip(outputs, want)):
            assert same(output, expected), f"call {place} of turn {turn}"


# rows x width: one CTA to a tile, and two to eight that share its K, at the tokens below
SHAPES = [(20000, 384), (9000, 640), (4608, 1024), (2048, 2048), (1024, 4608), (2048, 8192), (129, 1001), (40, 5000)]


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("tokens", [1, 2, 3, 7, 9, 15, 16, 17, 31, 33, 63, 65, 100, 127, 128])
def test_products_of_few_tokens(tokens, bits):
    calls = []
    status = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    for place, (rows, width) in enumerate(SHAPES):
        x, weight, gate = rows_of(tokens, width, bits, place), rows_of(rows, width, 4, 10 + place), rows_of(rows, width, 4, 20 + place)
        calls.append(lambda x=x, weight=weight: ops.linear_microscaled(x, weight, torch.float32, status=status))
        calls.append(lambda x=x, weight=weight: ops.linear_microscaled(x, weight, status=status))
        calls.append(lambda x=x, weight=weight, gate=gate: ops.gated_linear_microscaled(x, weight, gate, "silu", status=status))
    check_again(calls, 8)
    assert status.item() == 0


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("tokens,rows,width", [(129, 8192, 512), (333, 777, 1001), (700, 1700, 300), (1000, 520, 4000), (2049, 2048, 2048), (4000, 2048, 8192)])
def test_products_of_prompts(tokens, rows, width, bits):
    status = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    calls = []
    for seed in (1, 2):
        x, weight, gate = rows_of(tokens, width, bits, seed), rows_of(rows, width, 4, 10 + seed), rows_of(rows, width, 4, 20 + seed)
        calls.append(lambda x=x, weight=weight: ops.linear_microscaled(x, weight, torch.float32, status=status))
        calls.append(lambda x=x, weight=weight: ops.linear_microscaled(x, weight, status=status))
        calls.append(lambda x=x, weight=weight, gate=gate: ops.gated_linear_microscaled(x, weight, gate, "gelu", status=status))
    check_again(calls, 6)
    assert status.item() == 0


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("tokens,width", [(1, 32), (7, 1001), (130, 2048), (1000, 4608), (3000, 8192)])
def test_rows_and_norms(tokens, width, bits):
    calls = []
    for seed in (1, 2):
        generator = torch.Generator(device=DEVICE).manual_seed(seed)
        x, delta = (torch.randn(tokens, width, generator=generator, device=DEVICE) for _ in range(2))
        half, weight = delta.to(torch.bfloat16), 1 + 0.1 * torch.randn(width, generator=generator, device=DEVICE)
        calls.append(lambda x=x: ops.microscale(x, bits))
        calls.append(lambda half=half: ops.microscale(half, bits).values())
        calls.append(lambda x=x, half=half, weight=weight: ops.rmsnorm_microscaled(x, weight, 1e-5, delta=half, sum_out=torch.empty_like(x), bits=bits))
        calls.append(lambda x=x, delta=delta, weight=weight: ops.rmsnorm_microscaled(x, weight, 1e-5, delta=delta, bits=bits).values(torch.float32))
    check_again(calls, 10)


@pytest.mark.parametrize("tokens", [(20, 64), (33, 128), (100, 17), (1, 600)])
def test_beside_bfloat16_products(tokens):
    """Streams of bfloat16 and microscaled products in turn, K short and many tiles: all of them want tensor memory, and start early behind one another."""
    count, status = len(tokens), torch.zeros(1, dtype=torch.int32, device=DEVICE)
    x = [torch.randn(t, 256, device=DEVICE).to(torch.bfloat16) for t in tokens]
    weight, small = torch.randn(4096, 256, device=DEVICE).to(torch.bfloat16), rows_of(20000, 128, 4, 1)
    rows = [rows_of(t, 128, 8, t) for t in tokens]
    want = [(ops.linear(x[k], weight, status=status), ops.linear_microscaled(rows[k], small, status=status)) for k in range(count)]
    streams = [torch.cuda.Stream() for _ in range(count)]
    torch.cuda.synchronize()
    got = []
    for _ in range(40):
        for k, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got.append((k, ops.linear(x[k], weight, status=status), ops.linear_microscaled(rows[k], small, status=status)))
    torch.cuda.synchronize()
    assert status.item() == 0
    for k, one, other in got:
        assert torch.equal(one, want[k][0]) and torch.equal(other, want[k][1])
