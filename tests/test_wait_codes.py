"""What a wait that gave up is said to be: every code that the sources can leave has its role."""
import re
from pathlib import Path

import pytest
import torch

from gguf2bin_b200 import kernels_bf16
from gguf2bin_b200.kernels import KernelError

CSRC = Path(__file__).resolve().parent.parent / "gguf2bin_b200" / "csrc"
ROLES = {"PRODUCER": "the TMA producer", "MMA": "the MMA issuer", "ADDER": "an adder", "QUANTISER": "a quantising warp"}
LEFT = [(unit, role, int(code)) for unit in ("gemm_fp8_few", "gemm_fp8_tc")
        for role, code in re.findall(r"ST_(\w+)_TIMEOUT = (\d+)", (CSRC / f"{unit}.cuh").read_text())]


@pytest.mark.parametrize("unit,role,code", LEFT)
def test_codes_of_products_in_8_bits(unit, role, code, monkeypatch):
    monkeypatch.setattr(kernels_bf16, "_status", {torch.device("cpu"): torch.tensor([code], dtype=torch.int32)})
    with pytest.raises(KernelError, match=f"{unit} on cpu: {ROLES[role]} gave up"):
        kernels_bf16.check_status()
    kernels_bf16.check_status()                  # (the word is cleared)


def test_the_quantising_warps_have_a_code_of_their_own():
    text = (CSRC / "gemm_fp8_few.cuh").read_text()
    quantise = text[text.index("auto walk ="):text.index("if (p.x_f32) walk")]
    assert re.findall(r"ST_(\w+)_TIMEOUT", quantise) == ["QUANTISER"]
