"""``modules_to_not_convert`` of a routed model: all experts of a layer, or none of them."""
import pytest

import levolix_helpers as L
from gguf2bin_b200.config import model_spec_from_dict
from gguf2bin_b200.config.specs import ConfigError
from gguf2bin_b200.engine.model import expected_tensors
from test_eight_bit_models import FP8

CFG = L.CONFIGS["u"]


def config(*left_out):
    return dict(CFG, quantization_config=dict(FP8, modules_to_not_convert=list(left_out)))


def experts():
    """(the name of an expert's gate with a place for its number, the module that all experts are in)."""
    spec = model_spec_from_dict(config())
    i, layer = next((i, l) for i, l in enumerate(spec.layers) if l.feed_forward is not None and l.feed_forward.kind == "routed_experts")
    name = layer.prefix + dict(layer.feed_forward["names"])["gate"]
    name = name.removesuffix(".weight")
    return name, name[:name.index("{}")].rpartition(".")[0]


def test_one_expert_is_not_left_out():
    gate, before = experts()
    for name in (gate.format(0), gate.format(1), gate.format(0).rpartition(".")[0], gate.format(12)):
        with pytest.raises(ConfigError, match="not all matrices"):
            model_spec_from_dict(config(name))


def test_all_of_them_are():
    gate, before = experts()
    all_of = {n for n, e in expected_tensors(model_spec_from_dict(config())).items() if e.eight_bit}
    left = {n for n, e in expected_tensors(model_spec_from_dict(config(before, "lm_head", "no.such.module", before + ".x", before + "0"))).items() if e.eight_bit}
    assert left < all_of and all(n.startswith(before + ".") for n in all_of - left)
    assert gate.format(0) in all_of and gate.format(0) not in left
