"""Matrices in 8-bit floating point in a checkpoint: the tensors, their names, and how random ones are made.

A matrix ``name`` is F8_E4M3 [N, K]; ``name`` + "_scale_inv" holds the number that each block of 128 x 128 is multiplied with
(``csrc/fp8.cuh`` says how values are held)."""
from __future__ import annotations

import dataclasses

import torch

from .loader import Expected

F8 = torch.float8_e4m3fn
BLOCK = 128
MOST, LEAST = 448.0, 2.0 ** -100


def scale_name(name: str) -> str:
    return name + "_scale_inv"


def expect_eight_bit(expected: dict, names) -> dict:
    """``expected`` with the matrices ``names`` in 8 bits, each followed by its blocks' scales."""
    out = {}
    for name, e in expected.items():
        if name in names:
            out[name] = dataclasses.replace(e, eight_bit=True)
            out[scale_name(name)] = Expected(tuple(-(-int(n) // BLOCK) for n in e.shape), init="block_scales")
        else:
            out[name] = e
    return out


def held_on_cpu(w: torch.Tensor) -> tuple:
    """(entries [N, K], scales of the blocks) of a matrix: the operations of the CUDA kernel, one 32-bit rounding each."""
    n, k = w.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    full = torch.zeros(nb * BLOCK, kb * BLOCK, dtype=torch.float32)
    full[:n, :k] = w.float()
    tiles = full.view(nb, BLOCK, kb, BLOCK)
    m = tiles.abs().amax((1, 3)).clamp_min(LEAST)
    most = torch.full_like(m, MOST)
    q = (tiles * (most / m)[:, None, :, None]).reshape(nb * BLOCK, kb * BLOCK)[:n, :k].to(F8)
    return q.contiguous(), m / most


def held(w: torch.Tensor) -> tuple:
    """The same of a matrix wherever it is."""
    if not w.is_cuda:
        return held_on_cpu(w)
    from .. import kernels
    m = kernels.quantize_matrix(w)
    q = m.q if m.q.shape[1] == m.k else m.q.view(torch.uint8)[:, :m.k].contiguous().view(F8)
    return q, m.scale
