"""Weights that have just been brought back from microscaled rows, in products that ask for their weights before the kernel in front of them has ended."""

import pytest
import torch

from lalamo_b200 import ops

pytestmark = pytest.mark.gpu
DEVICE = "cuda"


def inputs(tokens, rows, width, bits):
    generator = torch.Generator(device=DEVICE).manual_seed(tokens + rows)
    x, others = (torch.randn(count, width, generator=generator, device=DEVICE).to(torch.bfloat16) for count in (tokens, rows))
    return x, others, ops.microscale(torch.randn(rows, width, generator=generator, device=DEVICE), bits)


@pytest.mark.parametrize("between", [False, True])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("tokens,rows,width", [(1, 2048, 8192), (16, 8192, 2048), (1, 17000, 1024), (17, 2048, 2048), (64, 2048, 4096), (128, 520, 1024), (200, 2048, 2048), (1000, 8192, 2048), (2048, 8192, 2048)])
def test_a_product_with_values(tokens, rows, width, bits, between):
    """Recorded, so that nothing but the kernels' order lies between the launches; what the values' place held before is not a number.  `between`: a product with other weights comes
    first, which lets its own successor start."""
    x, others, weight = inputs(tokens, rows, width, bits)
    want = ops.linear(x, weight.values().clone())
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.linear(x, others)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        values = weight.values()
        if between:
            ops.linear(x, others)
        out = ops.linear(x, values)
    for _ in range(20):
        values.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("tokens", [20, 100, 300, 2048])
def test_products_in_a_row(tokens):
    """As a user calls them: the values' place in memory is that of the weight before."""
    inputs_of = [inputs(tokens, 4096, 2048, bits) for bits in (8, 4)]
    want = []
    for x, _, weight in inputs_of:
        values = weight.values()
        torch.cuda.synchronize()
        want.append(ops.linear(x, values))
        del values
    torch.cuda.synchronize()
    got = [ops.linear(x, weight.values()) for _ in range(20) for x, _, weight in inputs_of]
    torch.cuda.synchronize()
    for place, out in enumerate(got):
        assert torch.equal(out, want[place % 2])


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("tokens", [1, 20, 64, 128, 200, 2048])
def test_every_kernel_reads_what_the_one_before_wrote(tokens, bits):
    """A chain in which each starts while the one before ends, recorded; before every replay all that lies between the first input and the last output is overwritten with
    what is no number."""
    generator = torch.Generator(device=DEVICE).manual_seed(tokens)
    width, hidden = 1024, 1536
    x = torch.randn(tokens, width, generator=generator, device=DEVICE).to(torch.bfloat16)
    weight = (torch.randn(width, width, generator=generator, device=DEVICE) / 32).to(torch.bfloat16)
    stream, scale = torch.randn(tokens, width, generator=generator, device=DEVICE), torch.ones(width, device=DEVICE)
    matrices = [torch.randn(*shape, generator=generator, device=DEVICE) / 32 for shape in ((hidden, width), (hidden, width), (width, hidden))]

    def chain():
        made = [ops.linear(x, weight)]
        total = torch.empty_like(stream)
        made.append(ops.rmsnorm_microscaled(stream, scale, 1e-5, delta=made[0], sum_out=total, bits=bits))
        made.append(total)
        up, gate, down = (ops.microscale(matrix, 4) for matrix in matrices)
        made += [up, gate, down, ops.gated_linear_microscaled(made[1], up, gate, "silu")]
        made.append(ops.linear_microscaled(made[-1], down))
        made.append(ops.microscale(made[-1], bits))
        made.append(made[-1].values())
        made.append(ops.linear_microscaled(made[-2], ops.microscale(weight, 4), torch.float32))
        return made

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    want = chain()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        made = chain()
    for _ in range(10):
        for one in made:
            if isinstance(one, ops.Microscaled):
                one.codes.fill_(255)
                one.scales.fill_(255)
            else:
                one.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for place, (one, expected) in enumerate(zip(made, want)):
            if isinstance(one, ops.Microscaled):
                assert torch.equal(one.codes, expected.codes) and torch.equal(one.values(torch.float32), expected.values(torch.float32)), place
            else:
                assert torch.equal(one, expected), place
