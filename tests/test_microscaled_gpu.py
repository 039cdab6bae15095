"""Microscaled rows (8 and 4 bits, a power of two per 32 columns) on the GPU against plain 64-bit arithmetic."""

import pytest
import torch

import plain_microscaled as plain
from lalamo_b200 import ops

pytestmark = pytest.mark.gpu
DEVICE = "cuda"


def activations(rows, width, seed, dtype=torch.float32):
    """Rows with channels of very different sizes, ties between two elements, empty blocks, signed zeros and numbers next to the type's ends."""
    generator = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, width, generator=generator) * torch.exp(2 * torch.randn(width, generator=generator))
    kind = torch.randint(0, 8, (rows, -(-width // 32)), generator=generator).repeat_interleave(32, dim=1)[:, :width]
    x = torch.where(kind == 0, torch.randint(-512, 513, (rows, width), generator=generator) / 16.0, x)  # many ties
    x = torch.where(kind == 1, 0.0 * x, x)  # zeros of both signs
    x = torch.where(kind == 2, x * 2.0**-122, x)  # scales at their lowest, subnormals in float32
    x = torch.where(kind == 3, (x.clamp(-60, 60) / 60) * 2.0**127, x)
    return x.to(dtype)


def made(rows: ops.Microscaled):
    """Codes and scale bytes of what a kernel made, on the CPU."""
    return plain.unpack(rows.codes.cpu(), rows.scales.cpu(), rows.bits)


def given(codes, scale_bytes, width, bits, rest=255):
    """Microscaled rows for the kernels, with scales that are not numbers behind the last row."""
    packed, scales = plain.pack(codes, scale_bytes, bits, rest)
    return ops.Microscaled(packed.to(DEVICE), scales.to(DEVICE), width, bits)


SIZES = [(1, 1), (1, 32), (3, 31), (5, 33), (130, 127), (129, 129), (7, 256), (300, 1001), (1, 8192), (33, 2048), (2, 40000)]


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,width", SIZES)
def test_microscale(rows, width, dtype, bits):
    """Every code and scale: the rule leaves nothing open."""
    x = activations(rows, width, 100 * rows + width, dtype)
    codes, scale_bytes = plain.quantise(x, bits)
    out = ops.microscale(x.to(DEVICE), bits)
    got_codes, got_bytes = made(out)
    assert torch.equal(got_bytes, scale_bytes)
    assert torch.equal(got_codes, codes)
    values = plain.stands_for(codes, scale_bytes, bits)[:, :width]
    assert torch.equal(out.values(torch.float32).cpu().double(), values)  # 4 significant bits, never below 2^-149
    assert torch.equal(out.values(torch.bfloat16).cpu(), values.to(torch.bfloat16))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_block_with_a_value_that_is_no_number(bad, bits):
    x = torch.randn(3, 200, generator=torch.Generator().manual_seed(1))
    x[1, 70] = bad
    out = ops.microscale(x.to(DEVICE), bits)
    values = out.values(torch.float32).cpu()
    want = plain.through(x, bits)
    assert torch.isnan(values[1, 64:96]).all() and torch.isnan(want[1, 64:96]).all()
    values[1, 64:96] = want[1, 64:96] = 0
    assert torch.equal(values.double(), want)


@pytest.mark.parametrize("bits", [8, 4])
def test_strange_addresses(bits):
    """Rows that do not start on 16 bytes."""
    x = activations(9, 264, 5)
    store = torch.empty(9 * 264 + 1, device=DEVICE)
    view = store[1:].view(9, 264)
    view.copy_(x)
    out = ops.microscale(view, bits)
    codes, scale_bytes = plain.quantise(x, bits)
    assert torch.equal(made(out)[0], codes) and torch.equal(made(out)[1], scale_bytes)


def between(got, one, other, slack=0.0):
    """Whether `got` lies between two bounds, element by element."""
    return bool(((got >= torch.minimum(one, other) - slack) & (got <= torch.maximum(one, other) + slack)).all())


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("delta", [None, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 31), (130, 128), (5, 1001), (2, 2048), (2, 2049), (3, 4104), (2, 8192), (1, 30001), (2, 32768)])
def test_norm(rows, width, delta, bits):
    """The sum is one rounding.  The norm's value is off by a few 2^-24 of itself for the factor (the sum of squares in float32: at most
    width additions of positive numbers, spread over 128 or more partial sums, below (width / 128 + 20) 2^-24; halved by the root) and two
    multiplications: less than 2^-15 for the widths here, so each quantised value lies between those of the 64-bit norm made smaller and larger by that."""
    generator = torch.Generator().manual_seed(rows + width)
    x = torch.randn(rows, width, generator=generator) * torch.exp(torch.randn(width, generator=generator))
    x[rows // 2] = 0
    d = None if delta is None else torch.randn(rows, width, generator=generator).to(delta)
    weight = 1 + 0.2 * torch.randn(width, generator=generator)
    total = x if d is None else x + d.float()
    sum_out = torch.full((rows, width), 7.0, device=DEVICE)
    out = ops.rmsnorm_microscaled(x.to(DEVICE), weight.to(DEVICE), 1e-5, delta=None if d is None else d.to(DEVICE), sum_out=sum_out, scale_offset=0.5, bits=bits)
    assert torch.equal(sum_out.cpu(), total)
    exact = total.double() / torch.sqrt(total.double().square().mean(dim=-1, keepdim=True) + 1e-5) * (weight.double() + 0.5)
    values = out.values(torch.float32).cpu().double()
    assert between(values, plain.through(exact * (1 - 2.0**-15), bits), plain.through(exact * (1 + 2.0**-15), bits))
    codes, _ = made(out)
    assert not codes[:, width:].any()


def test_norm_in_place_and_without_a_sum():
    generator = torch.Generator().manual_seed(3)
    x, d = torch.randn(5, 300, generator=generator), torch.randn(5, 300, generator=generator)
    weight = torch.ones(300, device=DEVICE)
    stream = x.to(DEVICE)
    first = ops.rmsnorm_microscaled(stream, weight, 1e-6, delta=d.to(DEVICE))
    assert torch.equal(stream.cpu(), x)
    second = ops.rmsnorm_microscaled(stream, weight, 1e-6, delta=d.to(DEVICE), sum_out=stream)
    assert torch.equal(stream.cpu(), x + d)
    assert torch.equal(first.codes, second.codes)
    third = ops.rmsnorm_microscaled(stream, weight, 1e-6)
    assert torch.equal(first.codes, third.codes)


def test_a_row_of_the_stream_that_is_no_number():
    x = torch.ones(3, 100)
    x[1, 5] = float("inf")
    values = ops.rmsnorm_microscaled(x.to(DEVICE), torch.ones(100, device=DEVICE), 1e-6).values().cpu()
    assert torch.isnan(values[1, :32]).all() and torch.isfinite(values[0]).all() and torch.isfinite(values[2]).all()


# ------------------------------------------------------------------------------------------------------------------ products


def whole_numbers(rows, width, bits, seed):
    """Codes whose values are small multiples of a half under scales of 1 to 8: sums of their products are exact in 32 bits whatever the order, so
    that a product has one right result and any scale, row or column out of place shows."""
    generator = torch.Generator().manual_seed(seed)
    columns = plain.padded(width)
    values = torch.randint(-4, 5, (rows, columns), generator=generator) / 2.0
    codes = torch.bucketize(values.abs().double(), plain.numbers(bits)) + (128 if bits == 8 else 8) * (values < 0)
    codes[:, width:] = 0
    scale_bytes = torch.randint(127, 131, (rows, columns // 32), generator=generator)
    return codes, scale_bytes, plain.stands_for(codes, scale_bytes, bits)


TOKENS = [1, 2, 8, 9, 16, 17, 33, 64, 65, 128, 129, 192, 193, 300, 385]


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("tokens", TOKENS)
@pytest.mark.parametrize("rows,width", [(128, 128), (129, 300), (1, 32), (777, 1001), (520, 2048), (8, 129), (264, 640)])
def test_product_of_whole_numbers(tokens, rows, width, bits):
    x_codes, x_bytes, x = whole_numbers(tokens, width, bits, tokens + width)
    w_codes, w_bytes, w = whole_numbers(rows, width, 4, rows + width)
    want = x @ w.T
    assert want.abs().max() < 2**24 / 4
    status = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    rows_given, weight_given = given(x_codes, x_bytes, width, bits), given(w_codes, w_bytes, width, 4)
    for dtype in (torch.float32, torch.bfloat16):
        got = ops.linear_microscaled(rows_given, weight_given, dtype, status=status)
        assert status.item() == 0
        assert torch.equal(got.cpu(), want.to(dtype)), f"{dtype}: {(got.cpu() != want.to(dtype)).sum().item()} of {want.numel()} differ"


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("tokens,rows,width", [(1, 2048, 8192), (8, 2048, 2048), (40, 1024, 4608), (333, 777, 1001), (1000, 512, 2048)])
def test_product_of_quantised_rows(tokens, rows, width, bits):
    """Sums of K products, exact each, in 32 bits: off by at most K 2^-23 of the sum of their sizes (an addition that cuts off instead of
    rounding loses up to 2^-23)."""
    x, w = activations(tokens, width, 3).clamp(-1e4, 1e4), torch.randn(rows, width, generator=torch.Generator().manual_seed(4)) * 0.02
    mine, weight = ops.microscale(x.to(DEVICE), bits), ops.microscale(w.to(DEVICE), 4)
    x, w = plain.through(x, bits), plain.through(w, 4)
    want, sizes = x @ w.T, x.abs() @ w.abs().T
    got = ops.linear_microscaled(mine, weight, torch.float32).cpu().double()
    assert bool(((got - want).abs() <= width * 2.0**-23 * sizes + 1e-40).all())
    # what one would see of a sum held in fewer bits: the errors of independent roundings are far below the bound
    assert (got - want).norm() <= 2.0**-18 * sizes.norm()
    rounded = ops.linear_microscaled(mine, weight).cpu()
    assert torch.equal(rounded, got.to(torch.bfloat16)) or tokens > 0 and between(rounded.double(), (got - width * 2.0**-23 * sizes).to(torch.bfloat16).double(), (got + width * 2.0**-23 * sizes).to(torch.bfloat16).double())


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("tokens", [1, 7, 16, 33, 65, 130, 200, 385])
@pytest.mark.parametrize("hidden,width", [(64, 128), (200, 300), (33, 1001), (264, 640), (1, 32)])
def test_gated_product_of_whole_numbers(tokens, hidden, width, bits):
    """The identity in place of an activation: up * gate, two whole numbers of halves below 2^12, is exact, and so is what comes out."""
    x_codes, x_bytes, x = whole_numbers(tokens, width, bits, tokens + width)
    keep = (torch.arange(plain.padded(width)) * 7 % max(1, plain.padded(width) // 16) == 0) | (torch.arange(plain.padded(width)) < 8)
    x_codes, x = torch.where(keep, x_codes, 0), torch.where(keep, x, 0.0)
    up_codes, up_bytes, up = whole_numbers(hidden, width, 4, 1)
    gate_codes, gate_bytes, gate = whole_numbers(hidden, width, 4, 2)
    u, g = x @ up.T, x @ gate.T
    assert torch.equal((u * g).float().double(), u * g)
    status = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    out = ops.gated_linear_microscaled(given(x_codes, x_bytes, width, bits), given(up_codes, up_bytes, width, 4), given(gate_codes, gate_bytes, width, 4), "identity", status=status)
    assert status.item() == 0
    assert (out.width, out.bits) == (hidden, 8)
    codes, scale_bytes = plain.quantise(u * g, 8)
    got_codes, got_bytes = made(out)
    assert torch.equal(got_bytes, scale_bytes)
    # a product of zero and a negative number is a negative zero, here and there alike
    assert torch.equal(got_codes, codes)


@pytest.mark.parametrize("activation,limit", [("silu", 0.0), ("gelu", 0.0), ("sigmoid_limit", 3.0)])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("tokens", [5, 150])
def test_gated_product(tokens, bits, activation, limit):
    """Values between those of the 64-bit result made smaller and larger by its error.  u and g are off by at most K 2^-23 of the sums of sizes S (see above);
    the activations here have slopes below 1.2 and are themselves off by less than 2^-20 of max(1, |g|) for |g| < 60 (float32 exp of an argument rounded by
    2^-24 |g|); so h is off by at most e = 1.3 (|u| + 1) K 2^-23 S_g + (|act(g)| + e_g) K 2^-23 S_u + 2^-19 (|u| + 1) max(1, |g|)."""
    hidden, width = 200, 512
    generator = torch.Generator().manual_seed(9)
    x = torch.randn(tokens, width, generator=generator)
    up, gate = (torch.randn(hidden, width, generator=generator) / width**0.5 * 3 for _ in range(2))
    out = ops.gated_linear_microscaled(ops.microscale(x.to(DEVICE), bits), ops.microscale(up.to(DEVICE), 4), ops.microscale(gate.to(DEVICE), 4), activation, limit=limit)
    x, up, gate = plain.through(x, bits), plain.through(up, 4), plain.through(gate, 4)
    u, g = x @ up.T, x @ gate.T
    error_u, error_g = (width * 2.0**-23 * (x.abs() @ w.abs().T) for w in (up, gate))
    assert g.abs().max() < 60
    h = plain.activate(g, u, activation, limit)
    error = 1.3 * (u.abs() + 1) * error_g + (1.2 * g.abs() + 1 + error_g) * error_u + 2.0**-19 * (u.abs() + 1) * g.abs().clamp(min=1)
    values = out.values(torch.float32).cpu().double()
    # the scale of a block may be the one above or below at a border; either rounding is within a step of the larger
    lower, upper = plain.through(h - error, 8), plain.through(h + error, 8)
    assert between(values, lower, upper)


def test_nothing_to_do():
    empty = ops.microscale(torch.empty(0, 300, device=DEVICE), 8)
    weight = ops.microscale(torch.randn(64, 300, device=DEVICE), 4)
    assert empty.values().shape == (0, 300)
    assert ops.linear_microscaled(empty, weight).shape == (0, 64)
    assert ops.gated_linear_microscaled(empty, weight, weight, "silu").shape == (0, 64)
    assert ops.linear_microscaled(ops.microscale(torch.randn(3, 300, device=DEVICE)), ops.microscale(torch.empty(0, 300, device=DEVICE), 4)).shape == (3, 0)
    assert ops.rmsnorm_microscaled(torch.empty(0, 300, device=DEVICE), torch.ones(300, device=DEVICE), 1e-5).shape == (0, 300)


@pytest.mark.parametrize("tokens", [3, 200])
def test_a_row_that_is_no_number_stays_in_its_row(tokens):
    x = torch.randn(tokens, 256, generator=torch.Generator().manual_seed(1))
    x[1, 3] = float("nan")
    weight = ops.microscale(torch.randn(130, 256, generator=torch.Generator().manual_seed(2)).to(DEVICE), 4)
    rows = ops.microscale(x.to(DEVICE))
    out = ops.linear_microscaled(rows, weight).cpu()
    others = torch.arange(tokens) != 1
    assert torch.isnan(out[1]).all() and torch.isfinite(out[others]).all()
    hidden = ops.gated_linear_microscaled(rows, weight, weight, "silu").values().cpu()
    assert torch.isnan(hidden[1]).all() and torch.isfinite(hidden[others]).all()


@pytest.mark.parametrize("tokens", [3, 200])
@pytest.mark.parametrize("activation", ["silu", "gelu", "sigmoid_limit"])
def test_activations_of_far_negative_gates(activation, tokens):
    """A block that has small values only has them as exactly as others.  Its gates g are one whole number down to -6, exact as the values of up are; the exponential of at most
    1.702 |g| is off by less than 2 + 1.2 * 1.702 |g| last places, erfc by 2 g^2 times the 2^-23 of its argument and 5 more, all of them below (g^2 + 12) 2^-23."""
    width = 128
    x = torch.zeros(tokens, width)
    x[:, 0] = 1.0
    up, gate = torch.zeros(96, width), torch.zeros(96, width)
    up[:, 0] = torch.tensor([1.0, 1.5, 2.0])[torch.arange(96) % 3]
    gate[:, 0] = -torch.tensor([6.0, 4.0, 3.0])[torch.arange(96) // 32]
    out = ops.gated_linear_microscaled(ops.microscale(x.to(DEVICE)), ops.microscale(up.to(DEVICE), 4), ops.microscale(gate.to(DEVICE), 4), activation, limit=7.0)
    g = gate[:, 0].double().expand(tokens, -1)
    h = plain.activate(g, up[:, 0].double().expand(tokens, -1), activation, 7.0)
    error = h.abs() * (g * g + 12) * 2.0**-23
    assert between(out.values(torch.float32).cpu().double(), plain.through(h - error, 8), plain.through(h + error, 8))


@pytest.mark.parametrize("tokens", [3, 200])
@pytest.mark.parametrize("activation", ["silu", "gelu", "sigmoid_limit", "identity"])
def test_no_activation_makes_a_number_of_what_is_none(activation, tokens):
    """Limits keep numbers within bounds; a NaN in `up` or in `gate` passes them."""
    generator = torch.Generator().manual_seed(5)
    x, w = torch.randn(tokens, 256, generator=generator), torch.randn(130, 256, generator=generator)
    x[1, 3] = float("nan")
    clean = ops.microscale(w.to(DEVICE), 4)
    hidden = ops.gated_linear_microscaled(ops.microscale(x.to(DEVICE)), clean, clean, activation, limit=3.0).values().cpu()
    others = torch.arange(tokens) != 1
    assert torch.isnan(hidden[1]).all() and torch.isfinite(hidden[others]).all()
    w[70, 200] = float("nan")
    weight, rows = ops.microscale(w.to(DEVICE), 4), ops.microscale(torch.randn(tokens, 256, generator=generator).to(DEVICE))
    for up, gate in ((weight, clean), (clean, weight)):
        hidden = ops.gated_linear_microscaled(rows, up, gate, activation, limit=3.0).values().cpu()
        assert torch.isnan(hidden[:, 64:96]).all() and torch.isfinite(hidden[:, :64]).all() and torch.isfinite(hidden[:, 96:]).all()


@pytest.mark.parametrize("tokens", [3, 200, 1000])
def test_a_weight_that_is_no_number_stays_in_its_rows(tokens):
    """Of the product in its column, of a gated product in its channel's block of 32."""
    generator = torch.Generator().manual_seed(4)
    w, x = torch.randn(200, 256, generator=generator), torch.randn(tokens, 256, generator=generator)
    w[70, 200] = float("inf")
    weight, rows, clean = ops.microscale(w.to(DEVICE), 4), ops.microscale(x.to(DEVICE)), ops.microscale(torch.randn(200, 256, generator=generator).to(DEVICE), 4)
    out = ops.linear_microscaled(rows, weight).cpu()
    assert torch.isnan(out[:, 70]).all() and torch.isfinite(out[:, :70]).all() and torch.isfinite(out[:, 71:]).all()
    for up, gate in ((weight, clean), (clean, weight)):
        hidden = ops.gated_linear_microscaled(rows, up, gate, "silu").values().cpu()
        assert torch.isnan(hidden[:, 64:96]).all() and torch.isfinite(hidden[:, :64]).all() and torch.isfinite(hidden[:, 96:]).all()


@pytest.mark.parametrize("tokens,rows", [(700, 1700), (4000, 520), (1030, 4608), (2500, 1000)])
@pytest.mark.parametrize("bits", [8, 4])
def test_many_tiles(tokens, rows, bits):
    """More tiles than multiprocessors, wide and narrow ones, the last cut short: whole numbers, so one right result."""
    x_codes, x_bytes, x = whole_numbers(tokens, 300, bits, tokens)
    w_codes, w_bytes, w = whole_numbers(rows, 300, 4, rows)
    want = (x.to(DEVICE) @ w.T.to(DEVICE))
    given_x, given_w = given(x_codes, x_bytes, 300, bits), given(w_codes, w_bytes, 300, 4)
    for dtype in (torch.float32, torch.bfloat16):
        assert torch.equal(ops.linear_microscaled(given_x, given_w, dtype), want.to(dtype))
    hidden = ops.gated_linear_microscaled(given_x, given_w, given_w, "identity")
    codes, scale_bytes = plain.quantise((want.float() * want.float()).cpu(), 8)   # both sides are exact in 32 bits, their product is rounded to them once
    got_codes, got_bytes = made(hidden)
    assert torch.equal(got_bytes, scale_bytes) and torch.equal(got_codes, codes)


@pytest.mark.parametrize("tokens,rows", [(393, 4931), (643, 4873)])
def test_tiles_of_two_multiprocessors(tokens, rows):
    """Rows of 8 bits and a K long enough for pairs of CTAs, an odd number of 128 rows of the weight, and a last tile of 73 tokens and of 3."""
    x_codes, x_bytes, x = whole_numbers(tokens, 8192, 8, tokens)
    w_codes, w_bytes, w = whole_numbers(rows, 8192, 4, rows)
    want = x.to(DEVICE) @ w.T.to(DEVICE)
    given_x, given_w = given(x_codes, x_bytes, 8192, 8), given(w_codes, w_bytes, 8192, 4)
    for dtype in (torch.float32, torch.bfloat16):
        assert torch.equal(ops.linear_microscaled(given_x, given_w, dtype), want.to(dtype))


def test_rows_past_4_gigabytes():
    """Elements, codes and outputs whose places need more than 32 bits: the last rows as in a call of their own."""
    rows, width = 67000, 65536
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device=DEVICE)
    x[-130:] = torch.randn(130, width, generator=torch.Generator().manual_seed(1)).to(DEVICE, torch.bfloat16)
    many, few = ops.microscale(x), ops.microscale(x[-130:].clone())
    assert torch.equal(many.codes[-130:], few.codes)
    values = many.values()
    assert torch.equal(values[-130:], few.values()) and not values[:-130].any()
    del values, x
    weight = ops.microscale(torch.randn(40, width, generator=torch.Generator().manual_seed(2)).to(DEVICE), 4)
    out = ops.linear_microscaled(many, weight, torch.float32)
    want = few.values(torch.float32).double() @ weight.values(torch.float32).double().T
    sizes = few.values(torch.float32).double().abs() @ weight.values(torch.float32).double().abs().T
    assert not out[:-130].any()
    assert bool(((out[-130:].double() - want).abs() <= width * 2.0**-23 * sizes).all())


# ------------------------------------------------------------------------------------------------------------------ together


def feed_forward(stream, delta, norm, up, gate, down, eps=1e-5):
    rows = ops.rmsnorm_microscaled(stream, norm, eps, delta=delta, sum_out=stream)
    return ops.linear_microscaled(ops.gated_linear_microscaled(rows, up, gate, "silu"), down)


def feed_forward_inputs(tokens, width, hidden, seed=0):
    generator = torch.Generator().manual_seed(seed)
    stream, delta = torch.randn(tokens, width, generator=generator), torch.randn(tokens, width, generator=generator).to(torch.bfloat16)
    norm = 1 + 0.1 * torch.randn(width, generator=generator)
    up, gate = (torch.randn(hidden, width, generator=generator) / width**0.5 for _ in range(2))
    return stream, delta, norm, up, gate, torch.randn(width, hidden, generator=generator) / hidden**0.5


@pytest.mark.parametrize("tokens,width,hidden", [(1, 256, 384), (9, 200, 328), (150, 256, 384), (400, 264, 700)])
def test_a_feed_forward(tokens, width, hidden):
    """The four together, weights quantised by the launches just before, against 64 bits with the same quantisations.  A value near a border may
    fall to the other side: a step of e4m3, 2^-3 of the value, in a few of some hundred terms; the bound leaves a hundredth of the result's size for it, and a
    half step for the rounding to bfloat16."""
    stream, delta, norm, up, gate, down = feed_forward_inputs(tokens, width, hidden)
    on_gpu = [t.to(DEVICE) for t in (stream, delta, norm, up, gate, down)]
    got = feed_forward(*on_gpu[:3], *(ops.microscale(w, 4) for w in on_gpu[3:])).cpu().double()
    total = stream + delta.float()
    assert torch.equal(on_gpu[0].cpu(), total)
    x = plain.through(total.double() / torch.sqrt(total.double().square().mean(dim=-1, keepdim=True) + 1e-5) * norm.double(), 8)
    h = plain.through(plain.activate(x @ plain.through(gate, 4).T, x @ plain.through(up, 4).T, "silu"), 8)
    want = h @ plain.through(down, 4).T
    assert (got - want).norm() <= (2.0**-8 + 0.01) * want.norm()


def test_recorded_and_replayed():
    """A recorded run gives, on new contents of the same tensors, what an eager one gives, bit for bit; twice the same."""
    stream, delta, norm, up, gate, down = (t.to(DEVICE) for t in feed_forward_inputs(12, 256, 384))
    weights = [ops.microscale(w, 4) for w in (up, gate, down)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        feed_forward(stream.clone(), delta, norm, *weights)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = feed_forward(stream, delta, norm, *weights)
    for seed in (1, 2):
        new_stream, new_delta = (t.to(DEVICE) for t in feed_forward_inputs(12, 256, 384, seed)[:2])
        stream.copy_(new_stream)
        delta.copy_(new_delta)
        graph.replay()
        first = out.clone()
        assert torch.equal(first, feed_forward(new_stream, new_delta, norm, *weights))
        stream.copy_(feed_forward_inputs(12, 256, 384, seed)[0])
        graph.replay()
        assert torch.equal(first, out)


def test_two_streams_at_once():
    inputs = [[t.to(DEVICE) for t in feed_forward_inputs(tokens, 512, 640, tokens)] for tokens in (5, 300)]
    weights = [[ops.microscale(w, 4) for w in one[3:]] for one in inputs]
    want = [feed_forward(one[0].clone(), *one[1:3], *w) for one, w in zip(inputs, weights)]
    streams = [torch.cuda.Stream() for _ in inputs]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for stream, one, w in zip(streams, inputs, weights):
            with torch.cuda.stream(stream):
                got.append(feed_forward(one[0].clone(), *one[1:3], *w))
    torch.cuda.synchronize()
    for k, out in enumerate(got):
        assert torch.equal(out, want[k % 2])
