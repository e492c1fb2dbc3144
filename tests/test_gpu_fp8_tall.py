"""Matrices in 8 bits of millions of rows: more tiles than a grid's second axis takes go to a kernel that takes them."""
from ctypes import addressof, c_int, c_longlong, c_void_p

import pytest
import torch

from fp8_plain import EPS, F8, held, rows_values
from test_gpu_kernels import DEV, rnd

pytestmark = pytest.mark.gpu


def test_every_choice_can_be_launched():
    """(The plans alone.)  Tiles of 128 rows of W, or of 64: at most 65,535 of either."""
    from gguf2bin_b200 import kernels_fp8 as K8
    size = K8._f("g2b_fp8_product_plan", [c_void_p, c_int, c_int])
    size.restype = c_longlong
    chosen = set()
    for N in (65535 * 64, 65535 * 64 + 16, 65535 * 128, 65535 * 128 + 16, 2 ** 24):
        for M in (*range(1, 40), 48, 64, 65, 100, 128, 129, 200, 300, 1000):
            for K in (64, 128, 1024):
                for epi in (K8.EPI_F32, K8.EPI_GATED_F32):
                    call = K8._Call()
                    call.M, call.N, call.K, call.epi, call.x_stride, call.ldw = M, N, K, epi, K, -(-K // 128) * 128
                    size(addressof(call), 1, 1)
                    chosen.add(call.columns)
                    assert call.columns == 0 or -(-N // (128 if call.columns > 0 else 64)) <= 65535, (M, N, K, call.columns)
    assert 0 in chosen and len(chosen) > 2


@pytest.mark.parametrize("M,N", [(3, 65535 * 128 + 40), (150, 65535 * 64 + 24)])
def test_products(M, N):
    from gguf2bin_b200 import kernels, kernels_bf16
    K = 128
    g = torch.Generator(device=DEV).manual_seed(1)
    q = torch.randint(0, 120, (N, K), generator=g, device=DEV, dtype=torch.uint8).view(F8)          # up to 2^8 (the largest are NaN's neighbours)
    w = kernels.Fp8Matrix(q, torch.rand(-(-N // 128), 1, generator=g, device=DEV) * 1e-3, K)
    x = rnd(M, K, seed=2, dtype=torch.bfloat16)
    out = torch.full((M, N), float("nan"), dtype=torch.bfloat16, device=DEV)
    kernels.linear(x, w, out)
    kernels_bf16.check_status()
    a = rows_values(*held(x))
    for at in (0, N // 2, N - 300):
        m = q[at:at + 300].double() * w.scale.cpu()[torch.arange(at, at + 300) // 128].double().to(DEV)
        ref, sums = a @ m.T, a.abs() @ m.abs().T
        # 128 products, each cut at 2^-23 of the largest at most, in 32-bit sums; bfloat16 behind it
        assert ((out[:, at:at + 300].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 132 * 4 * EPS * sums).all()
    assert not out.isnan().any()
