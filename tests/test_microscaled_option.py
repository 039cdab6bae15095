"""The engine's option for microscaled feed-forwards: which models have something that it holds so, which are refused, and the command-line flag."""

import pytest
import torch
from typer.testing import CliRunner

import tiny_mozetar
import tiny_tudulix
import tiny_vivulorn
import tiny_vuvulorn
import tiny_zevetar
import tiny_zozenex
from lalamo_b200.cli import app
from lalamo_b200.config import config_from_dict
from lalamo_b200.parts import Runtime
from lalamo_b200.parts.model import DecoderModel

FAMILIES = {"mozetar": tiny_mozetar, "tudulix": tiny_tudulix, "vivulorn": tiny_vivulorn, "vuvulorn": tiny_vuvulorn, "zevetar": tiny_zevetar, "zozenex": tiny_zozenex}
MODELS = [(family, name) for family, module in FAMILIES.items() for name in module.CONFIGS]


def gated(family, config):
    """Whether the configuration, as its family writes it, has a gated feed-forward of its own or beside routed experts."""
    for layer in config["layers"]:
        mlp = layer.get("mlp") or {}
        if family in ("vuvulorn", "zevetar") and mlp.get("kind") == "dense" or family in ("tudulix", "zevetar") and mlp.get("shared"):
            return True
    return False


def test_some_have_and_some_have_not():
    assert {family for family, name in MODELS if gated(family, FAMILIES[family].CONFIGS[name])} == {"tudulix", "vuvulorn", "zevetar"}
    assert not all(gated("tudulix", config) for config in tiny_tudulix.CONFIGS.values())


@pytest.mark.parametrize("family,name", MODELS)
def test_a_model_without_one_is_refused(family, name):
    """Before anything is built: without the tensors, a model that is taken misses one of them."""
    config = FAMILIES[family].CONFIGS[name]
    plan = config_from_dict(config).to_plan()
    runtime = Runtime(device=torch.device("cpu"), dtype=torch.bfloat16, microscaled_feed_forward=True)
    with pytest.raises((ValueError, KeyError)) as raised:
        DecoderModel(plan, {}, runtime)
    assert ("gated feed-forward" in str(raised.value)) == (not gated(family, config))
    with pytest.raises(KeyError):
        DecoderModel(plan, {}, Runtime(device=torch.device("cpu"), dtype=torch.bfloat16))


def test_the_flag(monkeypatch):
    from lalamo_b200.language_model import LanguageModel

    seen = []

    def made(preset, seed, **options):
        seen.append(options["engine_config"])
        raise ValueError("seen")

    monkeypatch.setattr(LanguageModel, "random", made)
    for flag in ([], ["--microscaled-feed-forward"]):
        result = CliRunner().invoke(app, ["generate", "--random-weights", "3", "--preset", "lfm2-1.2b", "--prompt-ids", "1 2", "--dtype", "bfloat16", *flag])
        assert result.exit_code != 0
    assert [config.microscaled_feed_forward for config in seen] == [False, True]


@pytest.mark.skipif(torch.cuda.is_available(), reason="without a device")
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("bits", [8, 4])
def test_which_kernel_without_a_device(bits, gated):
    from lalamo_b200 import ops

    for tokens in (1, 4096):
        with pytest.raises(ops.KernelError, match="device"):
            ops.microscaled_kernel(tokens, 2048, 8192, bits, gated)
    with pytest.raises(ops.KernelError, match="no kernel"):
        ops.microscaled_kernel(0, 2048, 8192, bits, gated)
