"""Products into a part of wider rows: what lies beside the outputs stays as it is, wherever their last column ends."""
import pytest
import torch

from gguf2bin_b200 import kernels_bf16


@pytest.mark.parametrize("dtype,step", [(torch.bfloat16, 8), (torch.float32, 4)])
@pytest.mark.parametrize("M,K", [(100, 4096), (300, 512), (2048, 4096), (4200, 512)])
def test_tiles_are_stored_only_where_the_columns_end_on_16_bytes(M, K, dtype, step, monkeypatch):
    monkeypatch.setattr(kernels_bf16, "_sm_count", lambda device: 148)
    base = torch.empty(M * 4128 + 16, dtype=dtype)
    first = -base.data_ptr() % 16 // base.element_size()
    wide = base[first:first + M * 4128].view(M, 4128)
    for n in range(4096 - step, 4097):
        tiles = kernels_bf16._tc_shape(M, n, wide[:, :n], K)[2] in (True, 2)
        assert tiles == (n % step == 0), n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", [(100, 2051, 2048), (300, 129, 256), (1100, 257, 4096), (1030, 2046, 4096), (4200, 1021, 512)])
def test_nothing_is_written_beside_the_outputs(M, N, K, dtype):
    """Every kernel of many rows: stored, added to, with an activation; outputs whose rows start on 16 bytes and end between them."""
    from gguf2bin_b200 import kernels
    from test_gpu_kernels import DEV, rnd
    a, w = rnd(M, K, dtype=torch.bfloat16, seed=1), rnd(N, K, dtype=torch.bfloat16, scale=0.1, seed=2)
    ref = a.double() @ w.double().T
    # 32-bit sums of K products of sizes that the reference has in the mean: K roundings of 2^-24 of the largest partial sum
    tol = K * 2.0 ** -24 * (a.double().abs() @ w.double().abs().T)
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    at = slice(16, 16 + N)
    wide = torch.full((M, -(-N // 8) * 8 + 32), 7.0, dtype=dtype, device=DEV)
    kernels.linear(a, w, wide[:, at])
    assert ((wide[:, at].double() - ref).abs() <= tol + half * (ref.abs() + tol)).all()
    assert (wide[:, :16] == 7).all() and (wide[:, 16 + N:] == 7).all()
    if dtype == torch.float32:
        wide = torch.full((M, -(-N // 8) * 8 + 32), -0.0, device=DEV)
        kernels.linear(a, w, wide[:, at], accumulate=True)
        assert ((wide[:, at].double() - ref).abs() <= tol + half * (ref.abs() + tol)).all()
        beside = torch.cat([wide[:, :16], wide[:, 16 + N:]], dim=1)
        assert not beside.any() and torch.signbit(beside).all()
    else:
        form = kernels.GluForm.gelu_tanh()
        wide = torch.full((M, -(-N // 8) * 8 + 32), 7.0, dtype=dtype, device=DEV)
        if kernels.linear_act(a, w, wide[:, at], form):
            want = torch.nn.functional.gelu(ref, approximate="tanh")
            # the activation's slope is at most 1.13; its own error is that of exp and a division in 32 bits, within 2^-18 of |z|
            assert ((wide[:, at].double() - want).abs() <= 1.2 * tol + half * (want.abs() + tol) + 2.0 ** -18 * ref.abs()).all()
            assert (wide[:, :16] == 7).all() and (wide[:, 16 + N:] == 7).all()
    kernels_bf16.check_status()
