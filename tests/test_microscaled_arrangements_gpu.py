"""Microscaled feed-forwards in every arrangement that has gated ones: norms on the sublayers' outputs, sublayers side by side, norms on both sides, a shared feed-forward beside
routed experts, a layer norm in front."""

import numpy as np
import pytest
import torch

import tiny_tudulix
import tiny_vuvulorn
import tiny_zevetar
from test_vuvulorn_gpu import run_schedule

from lalamo_b200 import ops
from lalamo_b200.config.plan import GatedMLPSpec, LayerNormSpec
from lalamo_b200.engine import Engine, EngineConfig
from lalamo_b200.parts import Runtime
from lalamo_b200.parts.base import build_part
from lalamo_b200.parts.block import PreNormBlock
from lalamo_b200.parts.feed_forward import GatedMLP

pytestmark = pytest.mark.gpu

MODELS = [
    ("vuvulorn", tiny_vuvulorn, "P"),  # norms on the outputs; a routed layer, one without a feed-forward, a gated one
    ("vuvulorn", tiny_vuvulorn, "Q"),
    ("tudulix", tiny_tudulix, "A"),  # norms on both sides; shared feed-forwards with limits
    ("zevetar", tiny_zevetar, "A"),  # side by side; gated ones, and shared ones under a gate
    ("zevetar", tiny_zevetar, "C"),
]


def by_operators(self, x, step=None, residual=None, defer=False):
    """A gated feed-forward as the operators make it, in an engine that knows nothing of them: weights quantised by every call, the result as a tensor."""
    up, gate = (ops.microscale(part.contiguous(), 4) for part in self.up_gate.chunk(2))
    hidden = ops.gated_linear_microscaled(ops.microscale(x, 8), up, gate, self.spec.activation, limit=self.spec.limit)
    out = ops.linear_microscaled(hidden, ops.microscale(self.down, 4))
    if residual is None:
        return out
    ops.residual_add(residual, out)
    return None


def gated_parts(engine):
    parts = [part for block in engine.model.blocks for part in block.parts()]
    parts += [sub for part in parts for sub in getattr(part, "sub_parts", list)()]
    return [part for part in parts if isinstance(part, GatedMLP)]


@pytest.mark.parametrize("family,module,name", MODELS, ids=lambda value: value if isinstance(value, str) else "")
def test_a_model_is_its_operators(family, module, name, tmp_path, monkeypatch):
    """The same bits as an engine whose gated feed-forwards are replaced, step by step without recordings: portions and single tokens, several requests."""
    config = module.CONFIGS[name]
    folder, _ = module.write_model(tmp_path / "model", config, 7)
    generator = np.random.default_rng(3)
    requests = {key: generator.integers(0, config["vocab"], size=count).tolist() for key, count in (("a", 70), ("b", 1), ("c", 200))}
    schedule = [[("a", 40), ("b", 1)], [("a", 1), ("c", 20)], [("a", 20), ("c", 150)]] + [[("a", 1), ("c", 1)]] * 9 + [[("c", 21)]]

    def made(**options):
        return Engine.load(folder, EngineConfig(dtype="bfloat16", page_size=16, max_tokens=1024, max_requests=4, cuda_graphs=False, poison_freed=True, **options))

    engine = made(microscaled_feed_forward=True)
    held = gated_parts(engine)
    assert held and all(part.takes_microscaled and not hasattr(part, "up_gate") for part in held)
    got = run_schedule(engine, requests, schedule)
    for key in requests:
        assert np.isfinite(got[key]).all()
    ordinary = made()
    assert len(gated_parts(ordinary)) == len(held)
    bfloat16 = run_schedule(ordinary, requests, schedule)
    monkeypatch.setattr(GatedMLP, "forward", by_operators)
    want = run_schedule(ordinary, requests, schedule)
    for key in requests:
        assert np.array_equal(got[key], want[key]), key
    assert any(not np.array_equal(bfloat16[key], want[key]) for key in requests)
    # recorded steps, which plan their attention otherwise, likewise
    recorded = {}
    for on in (True, False):
        if on:
            monkeypatch.undo()
        else:
            monkeypatch.setattr(GatedMLP, "forward", by_operators)
        replaying = Engine.load(folder, EngineConfig(dtype="bfloat16", page_size=16, max_tokens=1024, max_requests=4, poison_freed=True, microscaled_feed_forward=on))
        recorded[on] = run_schedule(replaying, requests, schedule)
    for key in requests:
        assert np.array_equal(recorded[True][key], recorded[False][key]), key


class Stub:
    """A mixer that hands on what it was given."""

    can_accumulate = False

    def __init__(self, out):
        self.out = out

    def forward(self, normed, step, cache):
        return self.out


@pytest.mark.parametrize("tokens", [1, 20, 300])
def test_a_layer_norm_in_front(tokens):
    """It hands out bfloat16 rows, which the feed-forward quantises."""
    runtime = Runtime(device=torch.device("cuda:0"), dtype=torch.bfloat16, microscaled_feed_forward=True)
    generator = torch.Generator().manual_seed(1)
    tensors = {name: torch.randn(*shape, generator=generator) / shape[1] ** 0.5 for name, shape in (("up_proj", (200, 96)), ("gate_proj", (200, 96)), ("down_proj", (96, 200)))}
    block = PreNormBlock.__new__(PreNormBlock)
    block.pre_mixer_norm, block.pre_ffn_norm = (
        build_part(LayerNormSpec(dim=96, eps=1e-5), {"scale": 1 + 0.1 * torch.randn(96, generator=generator), "bias": 0.1 * torch.randn(96, generator=generator)}, runtime) for _ in range(2)
    )
    mixed = torch.randn(tokens, 96, generator=generator).to("cuda", torch.bfloat16)
    block.mixer, block.ffn = Stub(mixed), build_part(GatedMLPSpec(model_dim=96, hidden_dim=200, activation="silu"), tensors, runtime)
    stream = torch.randn(tokens, 96, generator=generator).cuda()
    residual = stream.clone()
    out = block.forward(residual, None, None, None)
    assert torch.equal(residual, stream + mixed.float())
    rows = ops.microscale(block.pre_ffn_norm.forward(residual))
    up, gate, down = (ops.microscale(tensors[name].to("cuda", torch.bfloat16), 4) for name in ("up_proj", "gate_proj", "down_proj"))
    assert torch.equal(out, ops.linear_microscaled(ops.gated_linear_microscaled(rows, up, gate, "silu"), down))
    assert runtime.status.item() == 0
