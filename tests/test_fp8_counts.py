"""Counts beyond 32 bits are refused: the launchers would take them for others, or for nothing to do."""
import pytest
import torch

from fp8_plain import F8
from gguf2bin_b200 import kernels, kernels_fp8
from gguf2bin_b200.kernels import Fp8Matrix, Fp8Rows, KernelError

BIG = 2 ** 31


def meta(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")


def matrix(n, k, *lead, gated=False):
    kb = -(-k // 128)
    scales = (2, -(-n // 256), kb) if gated else (-(-n // 128), kb)
    return Fp8Matrix(meta(*lead, n, kb * 128, dtype=F8), meta(*lead, *scales), k)


@pytest.mark.parametrize("rows", [BIG, BIG + 5])
def test_rows(rows):
    with pytest.raises(KernelError, match="too many for one call"):
        kernels.quantize_rows(meta(rows, 4), Fp8Rows(meta(rows, 128, dtype=F8), meta(1, rows)))
    with pytest.raises(KernelError, match="too many for one call"):
        kernels.quantize_matrix(meta(rows, 4))
    with pytest.raises(KernelError, match="too many for one call"):
        kernels.linear(meta(rows, 4), matrix(8, 4), meta(rows, 8))
    with pytest.raises(KernelError, match="too many for one call"):
        kernels.linear(meta(8, 4), matrix(rows, 4), meta(8, rows))


@pytest.mark.parametrize("tokens,top", [(BIG, 1), (BIG // 2, 2), (BIG - 8192, 1), (2 ** 30, 4)])
def test_pairs(tokens, top):
    idx, pairs = meta(tokens, top, dtype=torch.int32), tokens * top
    pair_row = meta(pairs, dtype=torch.int32)
    with pytest.raises(KernelError, match="too many for one call"):
        kernels.moe_sort(idx, 4, meta(5, dtype=torch.int32), pair_row)
    with pytest.raises(KernelError, match="too many for one call"):
        kernels.moe_experts_fp8(meta(tokens, 8), idx, matrix(16, 8, 4, gated=True), matrix(4, 8, 4), meta(pairs, 4), pair_row)
    if pairs >= BIG:
        with pytest.raises(KernelError, match="too many for one call"):
            kernels.moe_back(meta(pairs, 4), pair_row, meta(tokens, top), meta(tokens, 4), meta(tokens, 4))


def test_the_largest_that_are_not():
    """(As far as the device, which there is none of.)"""
    idx = meta(BIG - 8193, 1, dtype=torch.int32)
    with pytest.raises(KernelError, match="CUDA"):
        kernels.moe_sort(idx, 4, meta(5, dtype=torch.int32), meta(BIG - 8193, dtype=torch.int32))
    assert kernels_fp8.SORTED_AT_ONCE == 8192
