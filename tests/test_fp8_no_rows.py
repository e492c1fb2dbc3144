"""Operators in 8-bit floating point of no tokens, and of tokens without choices."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent

PLAN = """
from ctypes import addressof, c_int, c_longlong, c_void_p
from gguf2bin_b200 import kernels_fp8 as K
call = K._Call()
call.M, call.top, call.n_experts, call.N, call.K, call.H, call.x_stride, call.ldw = {tokens}, {top}, 8, 128, 256, 256, 256, 256
size = K._f("g2b_fp8_experts_plan", [c_void_p, c_int, c_int])
size.restype = c_longlong
assert size(addressof(call), 1, 1) == 48          # the experts' first rows, on 16 bytes
"""


@pytest.mark.parametrize("tokens,top", [(0, 4), (0, 0), (5, 0)])
def test_the_plan_of_no_pairs(tokens, top):
    """(In a process of its own: a division by zero would end this one.)"""
    ran = subprocess.run([sys.executable, "-c", PLAN.format(tokens=tokens, top=top)], cwd=ROOT, capture_output=True, text=True)
    assert ran.returncode == 0, (ran.returncode, ran.stderr[-500:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,top", [(0, 4), (0, 0), (5, 0)])
def test_experts_of_no_pairs(tokens, top, dtype):
    from gguf2bin_b200 import kernels, kernels_bf16
    from test_gpu_fp8 import experts_case
    from test_gpu_kernels import DEV, rnd
    _, _, _, gu, down = experts_case(1, 1, 3, 0, 136, 256, 5)
    x = rnd(tokens, 256, seed=1).to(dtype)
    ints = lambda *shape: torch.full(shape, 9, dtype=torch.int32, device=DEV)
    rows, pair_row, weight = torch.empty(0, 256, device=DEV), ints(0), torch.empty(tokens, top, device=DEV)
    kernels.moe_experts_fp8(x, ints(tokens, top), gu, down, rows, pair_row)
    starts = ints(4)
    kernels.moe_sort(ints(tokens, top), 3, starts, pair_row)
    assert not starts.any()
    out = torch.full((tokens, 256), 3.0, dtype=dtype, device=DEV)
    kernels.moe_back(rows, pair_row, weight, x, out)
    assert not out.any()                                    # the sum of nothing
    acc = torch.full((tokens, 256), 3.0, device=DEV)
    kernels.moe_back(rows, pair_row, weight, x, acc, accumulate=True)
    assert (acc == 3).all()
    q = kernels.Fp8Rows(torch.empty(tokens, 256, dtype=torch.float8_e4m3fn, device=DEV), torch.empty(2, tokens, device=DEV))
    kernels.quantize_rows(x, q)
    kernels.quantize_rows(x, kernels.Fp8Rows(q.q[:0], q.scale[:, :0]), ints(tokens, 0))
    kernels_bf16.check_status()
    torch.cuda.synchronize()


def test_rows_without_places_are_written_nowhere():
    """Places [T, 0] have no address: nothing is launched for them (here, without a device, a launch is an error)."""
    from ctypes import c_int, c_longlong, c_void_p
    from gguf2bin_b200 import kernels_fp8 as K8
    f = K8._f("g2b_quantize_rows", [c_void_p, c_int, c_longlong, c_int, c_int, c_void_p, c_longlong, c_void_p, c_longlong, c_void_p, c_int, c_int, c_void_p])
    assert f(None, 0, 256, 5, 256, None, 256, None, 0, None, 0, 0, None) == 0
