"""Gated activations of values that are no numbers, or infinite: NaN where the gate or the up value is NaN, in every form and kernel."""
import math

import pytest
import torch

from fp8_plain import random_matrix
from test_gpu_fp8 import FORMS, new_rows
from test_gpu_kernels import DEV, rnd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", FORMS)
@pytest.mark.parametrize("M", [1, 9, 40, 150, 300])
def test_products_in_8_bits(M, name):
    """A row with a NaN is NaN throughout, as float and as quantised rows; the others have the bits that they have without it."""
    from gguf2bin_b200 import kernels
    I, K = 264, 384
    form = kernels.GluForm(*FORMS[name])
    w = kernels.Fp8Matrix(*random_matrix(I, K, DEV, 3, None, True), K)
    w = w._replace(scale=w.scale / math.sqrt(K))
    x = rnd(M, K, seed=M, dtype=torch.bfloat16)
    clean, out, odd = torch.empty(M, I, device=DEV), torch.full((M, I), 5.0, device=DEV), x.clone()
    odd[M // 2, 7] = math.nan
    rest = [i for i in range(M) if i != M // 2]
    kernels.gate_up_fused(x, w, clean, 8, form)
    kernels.gate_up_fused(odd, w, out, 8, form)
    assert out[M // 2].isnan().all() and torch.equal(out[rest], clean[rest]) and clean.isfinite().all()
    rows, as_clean = new_rows(M, I), new_rows(M, I)
    kernels.gate_up_fused(x, w, as_clean, 8, form)
    kernels.gate_up_fused(odd, w, rows, 8, form)
    assert rows.scale[:, M // 2].isnan().all() and rows.q[M // 2, :I].float().isnan().all()
    assert torch.equal(rows.q.view(torch.uint8)[rest], as_clean.q.view(torch.uint8)[rest]) and torch.equal(rows.scale[:, rest], as_clean.scale[:, rest])


@pytest.mark.parametrize("M", [1, 40, 300])
def test_gates_beyond_the_largest_number(M):
    """A gate that is infinite in 32 bits, SiLU: infinite times the up value, or no output of the gate below zero."""
    from gguf2bin_b200 import kernels
    I, K = 128, 128
    q, scale = random_matrix(I, K, DEV, 3, None, True)
    ones = torch.ones_like(q.float()).to(q.dtype)
    scale[0], scale[1] = 2e38, 1e-3
    x = torch.full((M, K), 4.0, device=DEV)
    out = torch.empty(M, I, device=DEV)
    kernels.gate_up_fused(x, kernels.Fp8Matrix(ones, scale, K), out, 8)
    assert (out == math.inf).all()
    kernels.gate_up_fused(-x, kernels.Fp8Matrix(ones, scale * torch.tensor([1e-30, 1.0], device=DEV)[:, None, None], K), out, 8)
    assert (out.abs() < 1e-30).all()


@pytest.mark.parametrize("name", FORMS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("block", [8, 12])
def test_gates_by_themselves(block, dtype, name):
    from gguf2bin_b200 import kernels
    I = 24
    z = rnd(6, I // block, 2, block, seed=1).to(dtype)
    form = kernels.GluForm(*FORMS[name])
    clean, out = torch.empty(6, I, dtype=dtype, device=DEV), torch.empty(6, I, dtype=dtype, device=DEV)
    kernels.swiglu(z.view(6, -1), clean, block, form=form)
    odd = z.clone()
    odd[1, 0, 0, 3], odd[2, 1, 1, 5] = math.nan, math.nan
    kernels.swiglu(odd.view(6, -1), out, block, form=form)
    assert out[1, 3].isnan() and out[2, block + 5].isnan() and int(out.isnan().sum()) == 2
    assert torch.equal(out[[0, 3, 4, 5]], clean[[0, 3, 4, 5]]) and clean.isfinite().all()
    if name == "silu":
        odd = z.clone()
        odd[1, 0, 0, 3], odd[1, 0, 1, 3] = math.inf, 2.0
        kernels.swiglu(odd.view(6, -1), out, block, form=form)
        assert out[1, 3] == math.inf


@pytest.mark.parametrize("name", ["gelu", "capped"])
@pytest.mark.parametrize("M", [4, 40, 200, 1100])
def test_products_in_bfloat16(M, name):
    from gguf2bin_b200 import kernels
    I, K = 256, 512
    w, x = rnd(2 * I, K, dtype=torch.bfloat16, scale=0.1, seed=1), rnd(M, K, dtype=torch.bfloat16, seed=2)
    x[M // 2, 5] = math.nan
    out = torch.empty(M, I, dtype=torch.bfloat16, device=DEV)
    assert kernels.gate_up_fused(x, w, out, 8, kernels.GluForm(*FORMS[name]))
    assert out[M // 2].isnan().all() and int(out.isnan().any(1).sum()) == 1
