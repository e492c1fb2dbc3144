"""What parts with matrices in 8-bit floating point share."""
from __future__ import annotations

import torch

from .. import kernels_fp8
from ..weights.eight_bit import F8, scale_name


def held_tensors(tensors: dict) -> dict:
    """``tensors`` with every matrix in 8 bits as ``kernels.Fp8Matrix`` (the scales stay there under their own names)."""
    return {name: kernels_fp8.stored_matrix(t, tensors[scale_name(name)]) if t.dtype == F8 else t for name, t in tensors.items()}


def flat_weights(*weights) -> list:
    """The tensors that matrices of either form, and other weights, consist of."""
    out = []
    for w in weights:
        if isinstance(w, torch.Tensor):
            out.append(w)
        elif isinstance(w, kernels_fp8.Fp8Matrix):
            out += [w.q, w.scale]
        elif isinstance(w, kernels_fp8.Fp8Matrices):
            out += [t for part in w.parts for t in (part.q, part.scale)]
    return out
