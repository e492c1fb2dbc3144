"""Matrices in 8 bits as a user makes them: from entries and scales, gate and up as one, stacks; and what the operators make of them."""
import pytest
import torch

from fp8_plain import F8, gate_up_values, held_matrix, matrix_values
from gguf2bin_b200 import kernels
from gguf2bin_b200.kernels import Fp8Matrix, KernelError


def stored(n, k, seed):
    q, s = held_matrix(torch.randn(n, k, generator=torch.Generator().manual_seed(seed)))
    return kernels.stored_matrix(q[:, :k], s)


def test_gate_and_up_and_stacks():
    gate, up = stored(136, 130, 1), stored(136, 130, 2)
    both = kernels.gate_up_matrix(gate, up)
    assert both.shape == (272, 130) and both.scale.shape == (2, 2, 2)
    for got, m in zip(gate_up_values(both.q, both.scale), (gate, up)):
        assert torch.equal(got, matrix_values(m.q, m.scale))
    three = kernels.stack_matrices(m for m in (both, both, both))
    assert three.shape == (3, 272, 130) and three.scale.shape == (3, 2, 2, 2) and torch.equal(three.q[1].view(torch.uint8), both.q.view(torch.uint8))


def test_refusals():
    gate, up = stored(136, 130, 1), stored(136, 130, 2)
    for a, b in ((gate, stored(128, 130, 2)), (gate, stored(136, 129, 2)), (stored(12, 130, 1), stored(12, 130, 2)),
                 (kernels.stack_matrices([gate, gate]), kernels.stack_matrices([up, up])), (kernels.gate_up_matrix(gate, up), kernels.gate_up_matrix(gate, up))):
        with pytest.raises(KernelError, match="gate_up_matrix"):
            kernels.gate_up_matrix(a, b)
    for bad in ([], [gate, stored(128, 130, 2)], [gate, stored(136, 129, 2)], [kernels.gate_up_matrix(gate, up), Fp8Matrix(stored(272, 130, 1).q, gate.scale, 130)],
                [kernels.stack_matrices([gate])]):
        with pytest.raises(KernelError, match="stack_matrices"):
            kernels.stack_matrices(bad)
    for q, s in ((gate.q, torch.ones(2, 1)), (gate.q.view(torch.uint8), torch.ones(2, 2)), (gate.q[None], torch.ones(2, 2)),
                 (gate.q, torch.ones(2, 2, dtype=torch.int32))):
        with pytest.raises(KernelError, match="stored_matrix"):
            kernels.stored_matrix(q, s)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 40, 300])
def test_from_matrices_to_experts(T):
    """Matrices quantised, put together and used: the bits of each expert by itself."""
    from test_gpu_kernels import DEV, rnd
    E, I, K, top = 3, 264, 320, 2
    gates, ups = ([rnd(I, K, scale=0.05, seed=10 * j + e) for e in range(E)] for j in (1, 2))
    gus = [kernels.gate_up_matrix(kernels.quantize_matrix(g), kernels.quantize_matrix(u)) for g, u in zip(gates, ups)]
    downs = [kernels.quantize_matrix(rnd(K, I, scale=0.05, seed=30 + e)) for e in range(E)]
    x = rnd(T, K, seed=4, dtype=torch.bfloat16)
    idx = torch.randint(0, E, (T, top), generator=torch.Generator().manual_seed(1)).to(torch.int32).to(DEV)
    rows, pair_row = torch.empty(T * top, K, device=DEV), torch.empty(T * top, dtype=torch.int32, device=DEV)
    kernels.moe_experts_fp8(x, idx, kernels.stack_matrices(gus), kernels.stack_matrices(downs), rows, pair_row)
    for e in range(E):
        token, choice = torch.nonzero(idx == e, as_tuple=True)
        if not len(token):
            continue
        mid, one = torch.empty(len(token), I, device=DEV), torch.empty(len(token), K, device=DEV)
        assert kernels.gate_up_fused(x[token].contiguous(), gus[e], mid, 8)
        kernels.linear(mid, downs[e], one)
        got = rows[pair_row.view(T, top)[token, choice].long()]
        # K in other parts may move a value between over a border of e4m3: 2^-3 of it, were it all of them
        assert (got - one).norm() <= 2.0 ** -3 * one.norm()
    assert gates[0].dtype == torch.float32 and downs[0].q.dtype == F8
