"""The gate of products in 8 bits that is left in float: 32 bits' precision, whichever kernel the number of rows gets."""
import math

import pytest
import torch

from fp8_plain import F8, held
from test_gpu_fp8 import FORMS
from test_gpu_kernels import DEV, rnd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", FORMS)
@pytest.mark.parametrize("columns", [0, 16, 32, 64, -64])
def test_gates_in_float(columns, name):
    """Where all blocks of gate and up have one scale the fused matrix is a plain one too, whose product in float, by the same kernel, holds the sums that
    the gate is made of.  From them on: exp within one step of 2^-23, and its argument off by half a step for each of its roundings (SiLU has none, the
    capped form a product, GELU three operations): both count as far as the exponential is not small beside one; the sum, the division, the
    product and up's offset half a step each."""
    from gguf2bin_b200 import kernels, kernels_bf16
    from gguf2bin_b200 import kernels_fp8 as K8
    M, I, K = 200, 264, 384
    form = kernels.GluForm(*(float(torch.tensor(v)) for v in FORMS[name]))
    g = torch.Generator(device=DEV).manual_seed(3)
    q = (60 * torch.randn(2 * I, K, generator=g, device=DEV)).clamp(-448, 448).to(F8)
    S = 2.0 ** -8
    rows = kernels.Fp8Rows(*held(rnd(M, K, seed=1) * torch.linspace(0.05, 3.0, M, device=DEV)[:, None]))
    sums, out = torch.empty(M, 2 * I, device=DEV), torch.empty(M, I, device=DEV)
    K8._product("test", rows, kernels.Fp8Matrix(q, torch.full((-(-2 * I // 128), 3), S, device=DEV), K), sums, K8.EPI_F32, columns=columns)
    K8._product("test", rows, kernels.Fp8Matrix(q, torch.full((2, -(-I // 128), 3), S, device=DEV), K), out, K8.EPI_GATED_F32, form=form, columns=columns)
    kernels_bf16.check_status()
    both = sums.double().view(M, I // 8, 2, 8)
    gate, up = both[:, :, 0].reshape(M, I).clamp_max(form.limit), both[:, :, 1].reshape(M, I).clamp(-form.limit, form.limit) + form.offset
    arg = gate * (form.c1 + form.c3 * gate * gate)
    want = gate * torch.sigmoid(arg) * up
    exp_share = torch.sigmoid(-arg)                              # of the exponential in the sum
    steps = (1 + {"silu": 0, "capped": 0.5, "gelu": 1.5}[name] * arg.abs()) * exp_share + 4 * 0.5
    near = arg > -80                                             # beyond, the quotient gets subnormal
    assert ((out.double() - want).abs() <= 1.01 * steps * 2.0 ** -23 * want.abs() + 1e-37)[near].all()
    assert (out[~near].double() - want[~near]).abs().max().item() < 1e-30 if (~near).any() else True
    assert (arg < -10).any() and gate.abs().max() > 5 if name == "silu" else math.isfinite(float(want.abs().max()))
