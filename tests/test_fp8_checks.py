"""Refusals of the operators in 8-bit floating point: wrong types, sizes, strides and devices are errors before anything is launched."""
import pytest
import torch

from fp8_plain import F8, held, held_matrix
from gguf2bin_b200 import kernels
from gguf2bin_b200.kernels import Fp8Matrix, Fp8Rows, KernelError


def rows(t, k, dtype=F8):
    kb = -(-k // 128)
    return Fp8Rows(torch.zeros(t, kb * 128, dtype=torch.uint8).view(F8) if dtype == F8 else torch.zeros(t, kb * 128, dtype=dtype), torch.zeros(kb, t))


def matrix(n, k, gated=False, stack=0):
    kb, lead = -(-k // 128), (stack,) if stack else ()
    scales = (2, -(-n // 256), kb) if gated else (-(-n // 128), kb)
    return Fp8Matrix(torch.zeros(*lead, n, kb * 128, dtype=torch.uint8).view(F8), torch.zeros(*lead, *scales), k)


def test_rows_are_checked():
    x = torch.zeros(3, 200)
    for bad in (Fp8Rows(rows(3, 200).q[:, :128], rows(3, 200).scale), Fp8Rows(rows(3, 200).q, torch.zeros(3, 2)),
                Fp8Rows(rows(3, 200).q, rows(3, 200).scale.double()), rows(3, 200, torch.uint8), rows(4, 200), rows(3, 300),
                Fp8Rows(torch.zeros(3, 264, dtype=torch.uint8).view(F8)[:, 8:], rows(3, 200).scale)):
        with pytest.raises(KernelError):
            kernels.quantize_rows(x, bad)
    with pytest.raises(KernelError, match="CUDA"):
        kernels.quantize_rows(x, rows(3, 200))
    with pytest.raises(KernelError, match="neighbouring"):
        kernels.quantize_rows(torch.zeros(200, 3).t(), rows(3, 200))
    with pytest.raises(KernelError, match="without values"):
        kernels.quantize_rows(torch.zeros(3, 0), rows(3, 1))
    with pytest.raises(KernelError, match="places"):
        kernels.quantize_rows(x, rows(6, 200), torch.zeros(3, 2, dtype=torch.int64))
    with pytest.raises(KernelError, match="places"):
        kernels.quantize_rows(x, rows(6, 200), torch.zeros(7, dtype=torch.int32))
    for bad in (torch.zeros(3), torch.zeros(4, 4).t(), torch.zeros(0, 4), torch.zeros(4, 4)):
        with pytest.raises(KernelError):
            kernels.quantize_matrix(bad)


def test_products_are_checked():
    x, w = torch.zeros(3, 200), matrix(50, 200)
    good = torch.zeros(3, 50)
    for a, m, out, kw in ((torch.zeros(3, 199), w, good, {}), (x, w, torch.zeros(3, 51), {}), (x, w, torch.zeros(4, 50), {}), (x, w, good.double(), {}),
                          (x, w, good.bfloat16(), dict(accumulate=True)), (x, w, torch.zeros(50, 3).t(), {}), (x, w._replace(k=100), good, {}),
                          (x, w._replace(scale=torch.zeros(2, 2)), good, {}), (x, w._replace(q=w.q.view(torch.uint8)), good, {}),
                          (x, w._replace(q=matrix(100, 200).q[::2]), good, {}), (rows(3, 300), w, good, {}), (rows(4, 200), w, good, {}),
                          (x, matrix(50, 200, stack=2), good, {}), (torch.zeros(3, 0), matrix(50, 0), good, {}), (x, w, torch.zeros(1, 50).expand(3, 50), {})):
        with pytest.raises(KernelError):
            kernels.linear(a, m, out, **kw)
    for a in (x, rows(3, 200)):
        with pytest.raises(KernelError, match="CUDA"):
            kernels.linear(a, w, good)


def test_gated_products_are_checked():
    x, w = torch.zeros(3, 200), matrix(48, 200, gated=True)
    for a, m, mid, block in ((x, w, torch.zeros(3, 24), 4), (x, w, torch.zeros(3, 24).bfloat16(), 8), (x, w, torch.zeros(3, 48), 8), (x, w, rows(4, 24), 8),
                             (x, w, rows(3, 200), 8), (x, matrix(40, 200, gated=True), torch.zeros(3, 20), 8), (x, matrix(48, 200), torch.zeros(3, 24), 8)):
        with pytest.raises(KernelError):
            kernels.gate_up_fused(a, m, mid, block)
    with pytest.raises(KernelError, match="CUDA"):
        kernels.gate_up_fused(x, w, torch.zeros(3, 24), 8)


def test_experts_are_checked():
    h, idx, gu, down = torch.zeros(3, 200), torch.zeros(3, 2, dtype=torch.int32), matrix(48, 200, True, 4), matrix(200, 24, stack=4)
    good, places = torch.zeros(6, 200), torch.zeros(6, dtype=torch.int32)
    for a, i, g, d, out in ((h, idx, gu, matrix(200, 25, stack=4), good), (h, idx, gu, matrix(200, 24, stack=3), good), (h, idx[:2], gu, down, good),
                            (h[:, :199], idx, gu, down, good), (h, idx, gu, down, good[:5]), (h, idx, gu, down, good.bfloat16()),
                            (h, idx, matrix(48, 200, True, 1025), matrix(200, 24, stack=1025), good)):
        with pytest.raises(KernelError):
            kernels.moe_experts_fp8(a, i, g, d, out, places)
    with pytest.raises(KernelError, match="CUDA"):
        kernels.moe_experts_fp8(h, idx, gu, down, good, places)
    for i, s, p in ((idx.long(), torch.zeros(5, dtype=torch.int32), places), (idx, torch.zeros(4, dtype=torch.int32), places),
                    (idx, torch.zeros(5, dtype=torch.int32), places[:5]), (idx, torch.zeros(5, dtype=torch.int32), places)):
        with pytest.raises(KernelError):
            kernels.moe_sort(i, 4, s, p)
    weight = torch.zeros(3, 2)
    for r, p, w, x, out, kw in ((good, places.long(), weight, h, h, {}), (good, places, weight.double(), h, h, {}), (good[:, :100], places, weight, h, h, {}),
                                (good, places, weight, h[:2], h, {}), (good, places, weight, h, h.bfloat16(), dict(accumulate=True)),
                                (good, places, weight, h, h, {})):
        with pytest.raises(KernelError):
            kernels.moe_back(r, p, w, x, out, **kw)


def test_matrices_put_together():
    from gguf2bin_b200 import kernels_fp8 as K
    g = torch.Generator().manual_seed(3)
    parts = [K.stored_matrix(*(lambda q, s: (q[:, :130], s))(*held_matrix(torch.randn(n, 130, generator=g)))) for n in (256, 128, 24)]
    assert parts[0].q.shape == (256, 256) and not parts[0].q.view(torch.uint8)[:, 130:].any()
    one = K.side_by_side(parts)
    assert isinstance(one, Fp8Matrix) and one.shape == (408, 130) and one.scale.shape == (4, 2)
    apart = K.side_by_side(parts[::-1])
    assert isinstance(apart, kernels.Fp8Matrices) and apart.shape == (408, 130) and apart.dtype == F8
    fused = K.gate_up_matrix(parts[0], parts[0])
    assert fused.scale.shape == (2, 2, 2) and torch.equal(fused.q.view(torch.uint8)[8:16], parts[0].q.view(torch.uint8)[:8])
    with pytest.raises(KernelError):
        K.gate_up_matrix(parts[0], parts[1])
    with pytest.raises(KernelError):
        K.stored_matrix(parts[0].q, torch.zeros(2, 1))
    assert K.stack_matrices([parts[0]] * 3).q.shape == (3, 256, 256)
    assert kernels.product_notices("x", one, torch.bfloat16) == [] and kernels.product_notices("x", apart, torch.bfloat16) == []


def test_the_plain_form_holds_what_it_says():
    x = torch.randn(5, 300, generator=torch.Generator().manual_seed(1))
    q, s = held(x)
    back = (q.double().view(5, 3, 128) * s.t().double()[:, :, None]).flatten(1)[:, :300]
    # half a step of three bits, 2^-4 of the value, or below the smallest normal value, 2^-6, half of 2^-9; and the 32-bit roundings
    assert ((back - x.double()).abs() <= torch.maximum(x.abs() * 2.0 ** -4, s.t().repeat_interleave(128, 1)[:, :300] * 2.0 ** -10) * (1 + 2.0 ** -20)).all()
