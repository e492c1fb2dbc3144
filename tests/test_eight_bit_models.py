"""Models with matrices in 8 bits, as far as no GPU is needed: configuration, tensors, loading, random weights."""
import json

import pytest
import torch

from fp8_plain import held_matrix
from gguf2bin_b200.config import model_spec_from_dict
from gguf2bin_b200.config.specs import ConfigError
from gguf2bin_b200.engine.model import expected_tensors
from gguf2bin_b200.weights import write_random_model
from gguf2bin_b200.weights.loader import Expected, load_weights
from gguf2bin_b200.weights.safetensors_io import WeightsError, write_safetensors

FP8 = dict(quant_method="fp8", fmt="e4m3", weight_block_size=[128, 128], activation_scheme="dynamic")
QWEN3 = dict(architectures=["Qwen3ForCausalLM"], hidden_size=192, intermediate_size=264, num_hidden_layers=2, num_attention_heads=4,
             num_key_value_heads=2, head_dim=64, vocab_size=311, rope_theta=1e6, rms_norm_eps=1e-6, tie_word_embeddings=True,
             max_position_embeddings=256)


def with_fp8(**more):
    return dict(QWEN3, quantization_config=dict(FP8, **more))


def test_the_matrices_of_a_qwen3_layer_are_expected_in_8_bits():
    exp, plain = expected_tensors(model_spec_from_dict(with_fp8())), expected_tensors(model_spec_from_dict(QWEN3))
    eight = {n for n, e in exp.items() if e.eight_bit}
    assert eight == {f"model.layers.{i}.{m}.weight" for i in (0, 1) for m in (
        "self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj", "self_attn.o_proj", "mlp.gate_proj", "mlp.up_proj", "mlp.down_proj")}
    assert set(exp) - set(plain) == {n + "_scale_inv" for n in eight}
    assert exp["model.layers.0.mlp.gate_proj.weight_scale_inv"].shape == (3, 2)
    assert exp["model.layers.1.self_attn.k_proj.weight_scale_inv"].shape == (1, 2)
    assert all(exp[n].shape == e.shape for n, e in plain.items())


def test_modules_may_be_left_out():
    exp = expected_tensors(model_spec_from_dict(with_fp8(modules_to_not_convert=["lm_head", "model.layers.0.mlp", "model.layers.1.self_attn.q_proj",
                                                                                 "model.layers.1.self_attn.k_proj", "model.layers.1.self_attn.v_proj",
                                                                                 "model.layers.1.self_attn.o_proj"])))
    eight = {n for n, e in exp.items() if e.eight_bit}
    assert not any(".0.mlp." in n or ".1.self_attn." in n for n in eight) and len(eight) == 7
    with pytest.raises(ConfigError, match="not all matrices"):
        model_spec_from_dict(with_fp8(modules_to_not_convert=["model.layers.0.mlp.up_proj"]))


@pytest.mark.parametrize("bad", [dict(quant_method="awq"), dict(fmt="e5m2"), dict(weight_block_size=[64, 128]), dict(weight_block_size=None),
                                 dict(activation_scheme="static"), dict(scale_fmt="ue8m0"), dict(group_size=32), dict(modules_to_not_convert="lm_head")])
def test_other_forms_are_refused(bad):
    with pytest.raises(ConfigError, match="quantization_config"):
        model_spec_from_dict(with_fp8(**bad))
    with pytest.raises(ConfigError):
        model_spec_from_dict(dict(QWEN3, quantization_config="fp8"))


def test_a_model_without_such_matrices_is_refused():
    from mopitar_helpers import CONFIGS
    name, cfg = next(iter(CONFIGS.items()))
    kinds = {p.kind for layer in model_spec_from_dict(cfg).layers for p in (layer.mixer, layer.feed_forward) if p is not None}
    spec = model_spec_from_dict(dict(cfg, quantization_config=FP8))
    eight = [n for n, e in expected_tensors(spec).items() if e.eight_bit]
    assert bool(eight) == bool(kinds & {"gqa_attention", "swiglu", "routed_experts"})
    with pytest.raises(ConfigError, match="no matrix"):
        every = [f"model.layers.{i}.{m}" for i in (0, 1) for m in ("mlp", "self_attn")]
        model_spec_from_dict(with_fp8(modules_to_not_convert=every))


def test_a_written_folder_holds_the_quantised_matrices(tmp_path):
    """The tensors of a folder in 8 bits are those of the same model without, quantised; the other tensors are what they were."""
    folder = write_random_model(tmp_path / "q", with_fp8(), 3, on_device=False)
    exp = expected_tensors(model_spec_from_dict(json.loads((folder / "config.json").read_text())))
    got = load_weights(folder, exp, torch.bfloat16, "cpu")
    from gguf2bin_b200.weights.random_init import random_tensor
    for i, (name, e) in enumerate(exp.items()):
        if e.optional or e.init == "block_scales":
            continue
        t = random_tensor(e, 3, i, torch.bfloat16, 0.02, 0.1)
        if e.eight_bit:
            q, scale = held_matrix(t)
            assert got[name].dtype == torch.float8_e4m3fn
            assert torch.equal(got[name].view(torch.uint8), q[:, :t.shape[1]].contiguous().view(torch.uint8)) and torch.equal(got[name + "_scale_inv"], scale)
        else:
            assert torch.equal(got[name], t)


def test_types_that_do_not_belong_are_one_error(tmp_path):
    f8 = torch.zeros(4, 4, dtype=torch.uint8).view(torch.float8_e4m3fn)
    write_safetensors(tmp_path / "model.safetensors", [("a", (4, 4), torch.float8_e4m3fn, lambda: f8), ("b", (4, 4), torch.bfloat16, lambda: torch.zeros(4, 4).bfloat16()),
                                                       ("b_scale_inv", (1, 1), torch.bfloat16, lambda: torch.ones(1, 1).bfloat16())])
    with pytest.raises(WeightsError, match="(?s)wrong type \\(2\\).* a  has unsupported dtype F8_E4M3.* b  has unsupported dtype BF16"):
        load_weights(tmp_path, {"a": Expected((4, 4)), "b": Expected((4, 4), eight_bit=True), "b_scale_inv": Expected((1, 1))}, torch.bfloat16, "cpu")
    got = load_weights(tmp_path, {"a": Expected((4, 4), eight_bit=True), "b": Expected((4, 4)), "b_scale_inv": Expected((1, 1))}, torch.float32, "cpu")
    assert got["a"].dtype == torch.float8_e4m3fn and got["b"].dtype == torch.float32


def test_a_mixer_binds_on_any_device():
    """Head gates fill the rows up to a multiple of eight: no kernel may run for that (the model's device need not be the current one)."""
    from mopitar_helpers import CONFIGS
    from gguf2bin_b200.kernels import Fp8Matrices, Fp8Matrix
    from gguf2bin_b200.parts.registry import mixer_class
    from gguf2bin_b200.weights.eight_bit import F8
    seen = 0
    for cfg in CONFIGS.values():
        spec = model_spec_from_dict(dict(cfg, quantization_config=FP8))
        for layer in spec.layers:
            if layer.mixer is None or not layer.mixer.get("eight_bit"):
                continue
            mixer = mixer_class(layer.mixer)(layer.mixer, spec.hidden_size, torch.float32, torch.device("cpu"))
            expected = mixer_class(layer.mixer).expected(layer.mixer, spec.hidden_size)
            mixer.bind({n: torch.ones(e.shape).to(F8) if e.eight_bit else torch.ones(e.shape) for n, e in expected.items()})
            rows = sum(e.shape[0] for n, e in expected.items() if e.eight_bit) - expected[mixer.names["o"]].shape[0]
            assert isinstance(mixer.w_qkv, (Fp8Matrix, Fp8Matrices)) and mixer.w_qkv.shape == (rows + -rows % 8, spec.hidden_size)
            seen += rows % 8 != 0
    assert seen
