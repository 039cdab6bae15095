"""Microscaled products of whole numbers, which have one right result, at the sizes where tiles are cut and shared out: gated ones cut in two, clusters of every size,
pairs of CTAs; and which kernel runs them."""

import pytest
import torch

import plain_microscaled as plain
from lalamo_b200 import ops
from test_microscaled_gpu import given, made, whole_numbers

pytestmark = pytest.mark.gpu
DEVICE = "cuda"


def check_product(tokens, rows, width, bits):
    x_codes, x_bytes, x = whole_numbers(tokens, width, bits, tokens + width)
    w_codes, w_bytes, w = whole_numbers(rows, width, 4, rows + width)
    want = x.to(DEVICE) @ w.T.to(DEVICE)
    assert want.abs().max() < 2**24 / 4
    given_x, given_w = given(x_codes, x_bytes, width, bits), given(w_codes, w_bytes, width, 4)
    status = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    for dtype in (torch.float32, torch.bfloat16):
        assert torch.equal(ops.linear_microscaled(given_x, given_w, dtype, status=status), want.to(dtype))
    assert status.item() == 0


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("tokens", [1, 7, 16, 17, 40, 64, 65, 128])
@pytest.mark.parametrize("hidden,width", [(8192, 2048), (4800, 300), (9400, 1001)])
def test_gated_products_cut_in_two(tokens, hidden, width, bits):
    """75 to 148 tiles of 64 rows of each weight: too many for the multiprocessors to share out, and cut in two all the same where K is long or the tokens are many.  Up times gate as
    in the tests of fewer tiles: few columns are not zero, so that the product of the two sums is exact."""
    assert 75 <= -(-hidden // 128) * 2 <= 148
    assert ops.microscaled_kernel(tokens, hidden, width, bits, gated=True) == "shared"
    columns = torch.arange(plain.padded(width))
    keep = (columns % 67 == 3) | (columns < 8)
    x_codes, x_bytes, x = whole_numbers(tokens, width, bits, tokens + width)
    x_codes, x = torch.where(keep, x_codes, 0), torch.where(keep, x, 0.0)
    up_codes, up_bytes, up = whole_numbers(hidden, width, 4, 1)
    gate_codes, gate_bytes, gate = whole_numbers(hidden, width, 4, 2)
    product = (x @ up.T) * (x @ gate.T)
    assert torch.equal(product.float().double(), product)
    status = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    out = ops.gated_linear_microscaled(given(x_codes, x_bytes, width, bits), given(up_codes, up_bytes, width, 4), given(gate_codes, gate_bytes, width, 4), "identity", status=status)
    assert status.item() == 0
    codes, scale_bytes = plain.quantise(product, 8)
    got_codes, got_bytes = made(out)
    assert torch.equal(got_bytes, scale_bytes) and torch.equal(got_codes, codes)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("tokens", [1, 5, 16, 31, 64, 100, 128])
@pytest.mark.parametrize("rows,width", [(20000, 500), (9000, 640), (6000, 1001), (4608, 2048), (3600, 2050), (3000, 2500), (2600, 3000), (2048, 8192)])
def test_clusters_of_every_size(tokens, rows, width, bits):
    """One tile a CTA, and two to eight CTAs to a tile; the tokens go round them, one of a cluster's CTAs with more than another."""
    assert ops.microscaled_kernel(tokens, rows, width, bits) == "shared"
    check_product(tokens, rows, width, bits)


@pytest.mark.parametrize("tokens,rows,width", [(4000, 3333, 8191), (2049, 8200, 8191), (4097, 4931, 6500)])
def test_pairs_of_ctas(tokens, rows, width):
    """Sizes that pairs run sooner by 7 % and more, by the costs that choose; odd numbers of rows, tokens and columns."""
    assert ops.microscaled_kernel(tokens, rows, width, 8) == "pairs"
    check_product(tokens, rows, width, 8)


def test_the_kernels():
    assert ops.microscaled_kernel(128, 100000, 8192, 8) == "shared"
    assert ops.microscaled_kernel(4096, 2048, 8192, 8) == "pairs"
    assert ops.microscaled_kernel(4096, 2048, 8192, 4) == "walked"   # pairs are for rows of 8 bits, and not for gated products
    assert ops.microscaled_kernel(4096, 2048, 8192, 8, gated=True) == "walked"
    assert ops.microscaled_kernel(4096, 2048, 128, 8) == "walked"
    assert ops.microscaled_kernel(500, 128, 8192, 8) == "shared"
    for sizes in ((0, 1, 1, 8), (1, 0, 1, 8), (1, 1, 0, 8), (1, 1, 1, 6)):
        with pytest.raises(ops.KernelError):
            ops.microscaled_kernel(*sizes)


def test_a_product_rounded_to_bfloat16():
    """The rounding of sums of quantised rows, by itself: off by at most half a step of the 32-bit sums, which the same call gives in float32."""
    generator = torch.Generator(device=DEVICE).manual_seed(3)
    for bits, tokens, rows, width in ((8, 8, 2048, 2048), (4, 333, 777, 1001), (8, 4096, 2048, 8192)):
        x, weight = ops.microscale(torch.randn(tokens, width, generator=generator, device=DEVICE), bits), ops.microscale(torch.randn(rows, width, generator=generator, device=DEVICE), 4)
        exact, rounded = ops.linear_microscaled(x, weight, torch.float32).double(), ops.linear_microscaled(x, weight).double()
        assert bool(((rounded - exact).abs() <= 2.0**-8 * exact.abs()).all())
        assert not torch.equal(rounded, exact)
