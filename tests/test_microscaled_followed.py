"""Microscaled operators refuse what somebody follows past them: tangents, function transforms, traces; and tensors without memory.  Nothing is launched then."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils.flop_counter import FlopCounterMode

from lalamo_b200 import ops
from test_microscaled import no_launch, on_cuda, rows  # noqa: F401


def calls(x, weight, delta):
    return {
        "microscale": lambda: ops.microscale(x),
        "norm": lambda: ops.rmsnorm_microscaled(x, weight, 1e-5),
        "norm with a delta": lambda: ops.rmsnorm_microscaled(x, weight, 1e-5, delta=delta, sum_out=x),
    }


def plain():
    return on_cuda(torch.zeros(3, 200)), on_cuda(torch.zeros(200)), on_cuda(torch.zeros(3, 200))


def products():
    x, weight = rows(3, 200, 8), rows(5, 200, 4)
    return {"values": lambda: x.values(), "product": lambda: ops.linear_microscaled(x, weight), "gated": lambda: ops.gated_linear_microscaled(x, weight, weight, "silu")}


def dual(tensor):
    made = torch.autograd.forward_ad.make_dual(tensor, torch.ones_like(tensor)).as_subclass(type(on_cuda(torch.zeros(1))))
    assert torch.autograd.forward_ad.unpack_dual(made.as_subclass(torch.Tensor)).tangent is not None
    return made


@pytest.mark.parametrize("place,name", [(0, "microscale"), (0, "norm"), (1, "norm"), (2, "norm with a delta")])
@pytest.mark.parametrize("gradients", [True, False])
def test_tangents(place, name, gradients):
    """Also without gradients: forward mode follows then too."""
    with torch.autograd.forward_ad.dual_level(), torch.set_grad_enabled(gradients):
        tensors = [torch.zeros(3, 200), torch.zeros(200), torch.zeros(3, 200)]
        tensors = [dual(tensor) if at == place else on_cuda(tensor) for at, tensor in enumerate(tensors)]
        with pytest.raises(ops.KernelError, match="backward|tangent"):
            calls(*tensors)[name]()
        with pytest.raises(AssertionError, match="launched"):   # plain tensors are nobody's, whatever the level
            calls(*plain())[name]()


def test_traces():
    def of(call):
        def traced(x):
            call()
            return x + 1

        return traced

    for call in {**calls(*plain()), **products()}.values():
        with pytest.raises(ops.KernelError, match="trace"):
            torch.jit.trace(of(call), torch.zeros(2))
        with pytest.raises(ops.KernelError, match="trace"):
            make_fx(of(call))(torch.zeros(2))
        with pytest.raises(AssertionError, match="launched"):   # counting is not following
            with FlopCounterMode(display=False):
                call()


def test_transforms():
    x, weight, delta = plain()

    def batched(scale):
        return ops.microscale((x * scale).as_subclass(type(x)))

    with pytest.raises(ops.KernelError):
        torch.func.vmap(batched)(torch.ones(4))
    with pytest.raises(ops.KernelError):
        torch.func.jvp(batched, (torch.ones(()),), (torch.ones(()),))


@pytest.mark.filterwarnings("ignore")
def test_tensors_without_memory(monkeypatch):
    with FakeTensorMode() as mode:
        x, weight = torch.empty(3, 200, device="cuda"), torch.empty(200, device="cuda")
        codes, scales = torch.empty(3, 256, dtype=torch.uint8, device="cuda"), torch.empty(1, 2, 512, dtype=torch.uint8, device="cuda")
        for call in (lambda: ops.microscale(x), lambda: ops.rmsnorm_microscaled(x, weight, 1e-5), lambda: ops.Microscaled(codes, scales, 200, 8).values()):
            with pytest.raises(ops.KernelError, match="memory"):
                call()
    for call in (lambda: ops.microscale(x), lambda: ops.rmsnorm_microscaled(x, weight, 1e-5), lambda: ops.Microscaled(codes, scales, 200, 8).values()):
        with pytest.raises(ops.KernelError, match="memory"):
            call()
    assert mode is not None
