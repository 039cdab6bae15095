"""Feed-forwards with weights of 4 bits and rows of 8 in the engine: the part against its operators, a small model against the plain implementation with the same
quantisations, recorded steps against eager ones."""

import numpy as np
import pytest
import torch

import plain_lfm2
import plain_microscaled as plain
from test_replay_gpu import RowChecker, bfloat16_limits
from tiny import TINY, make_model

from lalamo_b200 import ops
from lalamo_b200.config.plan import GatedMLPSpec, RMSNormSpec
from lalamo_b200.engine import Engine, EngineConfig, StepEntry
from lalamo_b200.parts import Runtime
from lalamo_b200.parts.base import build_part

pytestmark = pytest.mark.gpu


def through(rows, bits):
    return plain.through(rows, bits).to(rows.dtype)


def microscaled_swiglu(n2, w, prefix, rnd=plain_lfm2.exact):
    up, gate, down = (through(w[f"{prefix}.{name}.weight"], 4) for name in ("w3", "w1", "w2"))
    rows = through(n2, 8)
    return rnd(through(plain.activate(rows @ gate.T, rows @ up.T, "silu"), 8) @ down.T)


@pytest.fixture
def part():
    runtime = Runtime(device=torch.device("cuda:0"), dtype=torch.bfloat16, microscaled_feed_forward=True)
    generator = torch.Generator().manual_seed(1)
    tensors = {name: torch.randn(*shape, generator=generator) / shape[1] ** 0.5 for name, shape in (("up_proj", (200, 96)), ("gate_proj", (200, 96)), ("down_proj", (96, 200)))}
    return runtime, tensors, build_part(GatedMLPSpec(model_dim=96, hidden_dim=200, activation="silu"), tensors, runtime)


def test_the_part_is_its_operators(part):
    runtime, tensors, mlp = part
    up, gate, down = (ops.microscale(tensors[name].to("cuda", torch.bfloat16), 4) for name in ("up_proj", "gate_proj", "down_proj"))
    for tokens in (1, 20, 300):
        x = torch.randn(tokens, 96, device="cuda", dtype=torch.bfloat16)
        rows = ops.microscale(x)
        want = ops.linear_microscaled(ops.gated_linear_microscaled(rows, up, gate, "silu"), down)
        stream = torch.zeros(tokens, 96, device="cuda")
        for got in (mlp.forward(x), mlp.forward(rows), mlp.forward(x, defer=True), mlp.forward(x, residual=stream)):
            assert torch.equal(got, want)
        assert not stream.any()   # what is returned is not added
    assert runtime.status.item() == 0


def test_the_norm_in_front(part):
    """A product's sum in every form that a mixer leaves it in."""
    runtime, _, _ = part
    generator = torch.Generator().manual_seed(2)
    norm = build_part(RMSNormSpec(dim=96, eps=1e-5), {"scale": 1 + 0.1 * torch.randn(96, generator=generator)}, runtime)
    stream, slices = torch.randn(7, 96, generator=generator), torch.randn(3, 7, 96, generator=generator)
    plain_sum = slices.sum(0).to(torch.bfloat16)
    for delta, added in ((None, torch.zeros(7, 96)), (plain_sum.cuda(), plain_sum.float()), (ops.SlicedSum(slices.cuda(), torch.bfloat16), None)):
        residual = stream.cuda()
        rows = norm.residual_forward_microscaled(residual, delta)
        if added is None:
            expected = stream.cuda()
            ops.residual_add(expected, delta)
        else:
            expected = (stream + added).cuda()
        assert torch.equal(residual, expected)
        want = ops.rmsnorm_microscaled(expected, norm.scale, 1e-5)
        assert torch.equal(rows.codes, want.codes) and torch.equal(rows.values(), want.values())


@pytest.mark.parametrize("which", ["A", "C"])
def test_a_model(which, tmp_path, monkeypatch):
    """Prompts and decoded tokens, eager and recorded, against the plain model whose feed-forwards go through the same formats, within the limits that a plain run in
    bfloat16 gives; eager steps of two engines give the same bits.  (Recorded ones plan their attention for longer contexts, whose parts add up otherwise.)"""
    config, seed = TINY[which]
    monkeypatch.setattr(plain_lfm2, "swiglu", microscaled_swiglu)
    model_dir = make_model(tmp_path / "model", which)
    model = plain_lfm2.PlainModel(model_dir)
    generator = np.random.default_rng(50 + seed)
    sequences = [generator.integers(0, config["vocab_size"], size=n).tolist() for n in (40, 150, 230)]
    expected = [model.logits(tokens) for tokens in sequences]
    limits = bfloat16_limits(model, sequences, expected)
    decoded = 10
    seen = {}
    for graphs in (True, False, False):
        checker = RowChecker(limits)
        engine = Engine.load(model_dir, EngineConfig(dtype="bfloat16", max_tokens=1024, max_requests=4, cuda_graphs=graphs, microscaled_feed_forward=True))
        for index, (tokens, want) in enumerate(zip(sequences, expected)):
            head = len(tokens) - decoded
            engine.admit(index)
            got = engine.step([StepEntry(index, tokens[:head], list(range(head)))]).cpu()
            checker.add(got.numpy(), want[:head], f"prompt {index}")
            if not graphs:
                seen.setdefault((index, head), []).append(got)
        for place in range(decoded):
            got = engine.step([StepEntry(index, [tokens[len(tokens) - decoded + place]], [0]) for index, tokens in enumerate(sequences)]).cpu()
            want = torch.stack([want[len(tokens) - decoded + place] for tokens, want in zip(sequences, expected)])
            checker.add(got.numpy(), want, f"decoded token {place}")
            if not graphs:
                seen.setdefault(place, []).append(got)
        assert (engine.executor.graph_replays > 0) == graphs
        engine.executor.check_status()
        checker.finish()
    for one, other in seen.values():
        assert torch.equal(one, other)


def test_weights_are_held_once_and_small(tmp_path):
    model_dir = make_model(tmp_path / "model", "C")
    sizes = [Engine.load(model_dir, EngineConfig(max_tokens=256, max_requests=2, microscaled_feed_forward=on)).model.weight_bytes() for on in (False, True)]
    elements = 3 * 3 * 256 * 320   # of three layers' three matrices
    # up and gate, 320 x 256: 320 rows of 128 bytes and three tiles of 128 rows x two of 128 columns of scales; down, 256 rows of 192 bytes and two tiles x three
    held = 3 * (2 * (320 * 128 + 3 * 2 * 512) + 256 * 192 + 2 * 3 * 512)
    assert sizes[1] == sizes[0] - 2 * elements + held


def test_a_float32_engine_refuses(tmp_path):
    model_dir = make_model(tmp_path / "model", "A")
    with pytest.raises(ValueError, match="bfloat16"):
        Engine.load(model_dir, EngineConfig(dtype="float32", max_tokens=256, max_requests=2, microscaled_feed_forward=True))
