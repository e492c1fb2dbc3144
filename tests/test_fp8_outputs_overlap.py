"""Quantised rows whose scales lie on one another: refused where they are written, read as they are."""
import pytest
import torch

from gguf2bin_b200 import kernels
from gguf2bin_b200.kernels import Fp8Rows, KernelError
from test_fp8_checks import matrix, rows


@pytest.mark.parametrize("make", [lambda t: torch.zeros(1, t).expand(2, t), lambda t: torch.zeros(2 * t).as_strided((2, t), (t - 1, 1)),
                                  lambda t: torch.zeros(t + 1).as_strided((2, t), (1, 1))])
def test_scales_that_overlap(make):
    t = 3
    bad = Fp8Rows(rows(t, 200).q, make(t))
    with pytest.raises(KernelError, match="overlap"):
        kernels.quantize_rows(torch.zeros(t, 200), bad)
    with pytest.raises(KernelError, match="overlap"):
        kernels.quantize_rows(torch.zeros(1, 200), bad, torch.zeros(1, 3, dtype=torch.int32))
    with pytest.raises(KernelError, match="overlap"):
        kernels.gate_up_fused(torch.zeros(t, 200), matrix(2 * 200, 200, gated=True), bad, 8)
    # given rows are only read (here as far as the device, which there is none of)
    with pytest.raises(KernelError, match="CUDA"):
        kernels.linear(bad, matrix(50, 200), torch.zeros(t, 50))


def test_scales_that_do_not():
    """Rows of their own, wider ones, one block, one row."""
    for r in (rows(3, 200), Fp8Rows(rows(3, 200).q, torch.zeros(2, 8)[:, :3]), Fp8Rows(rows(3, 100).q, torch.zeros(1, 3).expand(1, 3)),
              Fp8Rows(rows(1, 200).q, torch.zeros(2, 1))):
        with pytest.raises(KernelError, match="CUDA"):
            kernels.quantize_rows(torch.zeros(r.q.shape[0], 200 if r.scale.shape[0] == 2 else 100), r)
