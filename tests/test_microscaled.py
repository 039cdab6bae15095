"""What the microscaled operators refuse, and that nothing is launched then."""

import pytest
import torch

import plain_microscaled as plain
from lalamo_b200 import ops


class _NoLaunch:
    def __getattr__(self, name):
        raise AssertionError(f"{name} was launched")


class _OnCuda(torch.Tensor):
    """A tensor that says that it lies on a device of a certain number."""

    is_cuda = True
    device_number = 0

    def get_device(self):
        return self.device_number

    @classmethod
    def __torch_function__(cls, function, types, arguments=(), keywords=None):
        with torch._C.DisableTorchFunctionSubclass():
            return function(*arguments, **(keywords or {}))


def on_cuda(tensor, device=0):
    tensor = tensor.as_subclass(_OnCuda)
    tensor.device_number = device
    return tensor


def aligned(*shape):
    """Zeros that start on 64 bytes."""
    count = 1
    for size in shape:
        count *= size
    store = torch.zeros(count + 64, dtype=torch.uint8)
    first = -store.data_ptr() % 64
    return store[first : first + count].view(shape)


def rows(count, width, bits, changed=None):
    columns = plain.padded(width)
    fields = {"codes": on_cuda(aligned(count, columns * bits // 8)), "scales": on_cuda(aligned(-(-count // 128), columns // 128, 512)), "width": width, "bits": bits}
    return ops.Microscaled(**{**fields, **(changed or {})})


@pytest.fixture(autouse=True)
def no_launch(monkeypatch):
    monkeypatch.setattr(ops, "_lib", lambda: _NoLaunch())
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "_current_device", lambda: 0)


def test_the_stand_ins_reach_the_launch():
    """What the refusals below change one thing of is taken."""
    with pytest.raises(AssertionError, match="lb_gemm_microscaled"):
        ops.linear_microscaled(rows(3, 200, 8), rows(5, 200, 4))
    with pytest.raises(AssertionError, match="lb_gated_microscaled"):
        ops.gated_linear_microscaled(rows(3, 200, 4), rows(5, 200, 4), rows(5, 200, 4), "silu")
    with pytest.raises(AssertionError, match="lb_microscaled_values"):
        rows(3, 200, 8).values()


@pytest.mark.parametrize(
    "bad",
    [
        {"bits": 6},
        {"width": 0},
        {"width": 300},  # three blocks of 128
        {"codes": on_cuda(aligned(3, 128))},
        {"codes": on_cuda(aligned(3 * 256))},
        {"codes": on_cuda(aligned(3, 512)[:, ::2])},
        {"codes": on_cuda(torch.zeros(3, 256, dtype=torch.int8))},
        {"scales": on_cuda(aligned(2, 2, 512))},
        {"scales": on_cuda(aligned(1, 1, 512))},
        {"scales": on_cuda(aligned(1, 2, 256))},
        {"codes": on_cuda(aligned(3, 256), device=1)},
        {"scales": on_cuda(aligned(1, 2, 512), device=1)},
        {"codes": aligned(3, 256)},
        {"scales": aligned(1, 2, 512)},
        {"codes": on_cuda(aligned(3 * 256 + 16)[16:].view(3, 256))},  # starts on 16 bytes
        {"scales": on_cuda(aligned(1024 + 8)[8:].view(1, 2, 512))},
    ],
    ids=str,
)
def test_rows_that_are_none(bad):
    with pytest.raises(ops.KernelError):
        rows(3, 200, 8, bad)


def test_rows_on_another_device(monkeypatch):
    one, weight = rows(3, 200, 8), rows(5, 200, 4)
    elsewhere = ops.Microscaled(on_cuda(aligned(5, 128), device=1), on_cuda(aligned(1, 2, 512), device=1), 200, 4)
    for call in (
        lambda: ops.linear_microscaled(one, elsewhere),
        lambda: ops.linear_microscaled(elsewhere, weight),
        lambda: ops.gated_linear_microscaled(one, weight, elsewhere, "silu"),
        lambda: ops.gated_linear_microscaled(one, elsewhere, weight, "silu"),
        lambda: ops.linear_microscaled(one, weight, status=on_cuda(torch.zeros(1, dtype=torch.int32), device=1)),
        lambda: elsewhere.values(),
    ):
        with pytest.raises(ops.KernelError, match="device"):
            call()


def test_products_that_do_not_fit():
    for x, weight in ((rows(3, 200, 8), rows(5, 201, 4)), (rows(3, 200, 8), rows(5, 200, 8)), (rows(3, 200, 8), rows(5, 72, 4))):
        with pytest.raises(ops.KernelError):
            ops.linear_microscaled(x, weight)
        for up, gate in ((weight, rows(5, 200, 4)), (rows(5, 200, 4), weight)):
            with pytest.raises(ops.KernelError):
                ops.gated_linear_microscaled(x, up, gate, "silu")
    good = rows(5, 200, 4)
    with pytest.raises(ops.KernelError):
        ops.linear_microscaled(rows(3, 200, 8), good, torch.float16)
    with pytest.raises(ops.KernelError):
        ops.linear_microscaled(rows(3, 200, 8), good, status=torch.zeros(1))
    with pytest.raises(ops.KernelError):
        ops.gated_linear_microscaled(rows(3, 200, 8), good, rows(6, 200, 4), "silu")
    with pytest.raises(ops.KernelError):
        ops.gated_linear_microscaled(rows(3, 200, 8), good, good, "tanh")
    with pytest.raises(ops.KernelError):
        ops.gated_linear_microscaled(rows(3, 200, 8), rows(0, 200, 4), rows(0, 200, 4), "silu")


def test_rows_to_quantise():
    good = on_cuda(torch.zeros(3, 200))
    with pytest.raises(AssertionError, match="lb_microscale"):
        ops.microscale(good)
    for x, bits in (
        (good, 6),
        (torch.zeros(3, 200), 8),
        (on_cuda(torch.zeros(3, 200), device=1), 8),
        (on_cuda(torch.zeros(200)), 8),
        (on_cuda(torch.zeros(2, 3, 200)), 8),
        (on_cuda(torch.zeros(3, 0)), 8),
        (on_cuda(torch.zeros(3, 400)[:, ::2]), 8),
        (on_cuda(torch.zeros(3, 200, dtype=torch.float16)), 8),
        (on_cuda(torch.zeros(3, 200, dtype=torch.float64)), 8),
    ):
        with pytest.raises(ops.KernelError):
            ops.microscale(x, bits)


def test_norms():
    x, weight = on_cuda(torch.zeros(3, 200)), on_cuda(torch.zeros(200))
    with pytest.raises(AssertionError, match="lb_rmsnorm_microscaled"):
        ops.rmsnorm_microscaled(x, weight, 1e-5, delta=on_cuda(torch.zeros(3, 200)), sum_out=x)
    store = torch.zeros(700)
    for changed in (
        {"x": on_cuda(torch.zeros(3, 200, dtype=torch.bfloat16))},
        {"x": on_cuda(torch.zeros(600))},
        {"x": torch.zeros(3, 200)},
        {"x": on_cuda(torch.zeros(3, 200), device=1)},
        {"weight": on_cuda(torch.zeros(201))},
        {"weight": on_cuda(torch.zeros(200, dtype=torch.bfloat16))},
        {"weight": on_cuda(torch.zeros(200), device=1)},
        {"weight": on_cuda(torch.zeros(1, 200))},
        {"bits": 6},
        {"delta": on_cuda(torch.zeros(2, 200))},
        {"delta": on_cuda(torch.zeros(3, 200, dtype=torch.float16))},
        {"delta": on_cuda(torch.zeros(3, 200), device=1)},
        {"sum_out": on_cuda(torch.zeros(3, 200, dtype=torch.bfloat16))},
        {"sum_out": on_cuda(torch.zeros(4, 200))},
        {"sum_out": on_cuda(torch.zeros(3, 200), device=1)},
        {"x": on_cuda(store[:600].view(3, 200)), "sum_out": on_cuda(store[100:].view(3, 200))},
        {"delta": on_cuda(store[:600].view(3, 200)), "sum_out": on_cuda(store[:600].view(3, 200))},
        {"weight": on_cuda(store[500:]), "sum_out": on_cuda(store[:600].view(3, 200))},
        {"x": on_cuda(torch.zeros(1, 32769)), "weight": on_cuda(torch.zeros(32769))},
    ):
        arguments = {"x": x, "weight": weight, "eps": 1e-5, **changed}
        with pytest.raises(ops.KernelError):
            ops.rmsnorm_microscaled(**arguments)


def test_the_plain_implementation():
    """Against torch's own e4m3, and by hand for e2m1."""
    x = torch.randn(5, 64, generator=torch.Generator().manual_seed(1)) * 3
    scaled = x.view(5, 2, 32) / 2.0 ** (torch.frexp(x.view(5, 2, 32).abs().amax(-1)).exponent - 9)[..., None]
    want = scaled.clamp(-448, 448).to(torch.float8_e4m3fn)
    codes, _ = plain.quantise(x, 8)
    assert torch.equal(codes[:, :64].to(torch.uint8), want.view(torch.uint8).view(5, 64))
    row = torch.zeros(1, 32)
    row[0, :10] = torch.tensor([7.0, 5.0, -5.1, 0.25, 0.26, -0.75, 1.25, 1.75, 2.5, 3.5])
    codes, scale_bytes = plain.quantise(row, 4)
    assert scale_bytes[0, 0] == 127
    assert codes[0, :10].tolist() == [7, 6, 15, 0, 1, 10, 2, 4, 4, 6]
    for bits in (8, 4):
        codes, scale_bytes = plain.quantise(torch.randn(130, 300), bits)
        back = plain.unpack(*plain.pack(codes, scale_bytes, bits), bits)
        assert torch.equal(back[0], codes) and torch.equal(back[1], scale_bytes)


def test_tensors_that_autograd_follows():
    x, weight = on_cuda(torch.zeros(3, 200)), on_cuda(torch.zeros(200))
    followed, followed_weight = on_cuda(torch.zeros(3, 200)).requires_grad_(), on_cuda(torch.zeros(200)).requires_grad_()
    with pytest.raises(ops.KernelError, match="backward"):
        ops.microscale(followed)
    for changed in ({"x": followed}, {"weight": followed_weight}, {"delta": followed}):
        with pytest.raises(ops.KernelError, match="backward"):
            ops.rmsnorm_microscaled(**{"x": x, "weight": weight, "eps": 1e-5, **changed})
    with torch.no_grad(), pytest.raises(AssertionError, match="lb_microscale"):
        ops.microscale(followed)
