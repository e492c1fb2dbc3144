"""The scales of a checkpoint's blocks: 32 bits wide, whatever type of floating point they are stored in; no other types."""
import pytest
import torch

from gguf2bin_b200.weights.loader import Expected, load_weights
from gguf2bin_b200.weights.safetensors_io import WeightsError, write_safetensors

EXPECTED = {"w": Expected((130, 4), eight_bit=True), "w_scale_inv": Expected((2, 1), init="block_scales")}


def folder(path, scale):
    f8 = torch.zeros(130, 4, dtype=torch.uint8).view(torch.float8_e4m3fn)
    write_safetensors(path / "model.safetensors", [("w", (130, 4), torch.float8_e4m3fn, lambda: f8), ("w_scale_inv", (2, 1), scale.dtype, lambda: scale)])
    return path


@pytest.mark.parametrize("compute", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("stored", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
def test_scales_keep_their_values(tmp_path, stored, compute):
    scale = torch.tensor([[1 + 2.0 ** -10], [0.0123456789]]).to(stored)
    got = load_weights(folder(tmp_path, scale), EXPECTED, compute, "cpu")
    assert got["w_scale_inv"].dtype == torch.float32 and torch.equal(got["w_scale_inv"], scale.float())


@pytest.mark.parametrize("stored", [torch.int32, torch.uint8, torch.int64, torch.bool])
def test_scales_of_other_types_are_refused(tmp_path, stored):
    with pytest.raises(WeightsError, match="w_scale_inv  has unsupported dtype"):
        load_weights(folder(tmp_path, torch.ones(2, 1, dtype=stored)), EXPECTED, torch.float32, "cpu")
