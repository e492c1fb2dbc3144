"""Products in 8 bits behind a kernel that lets them in early and takes far longer than their waits are bounded by: the waits begin when it has ended."""
import pytest
import torch

from fp8_plain import held
from test_gpu_fp8 import operands
from test_gpu_kernels import DEV

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("columns,split", [("given", 0), ("on the way", 2), (16, 3), (32, 1), (64, 2), (-64, 4), (0, 1)])
def test_waits_begin_behind_it(columns, split):
    from gguf2bin_b200 import kernels, kernels_bf16
    from gguf2bin_b200 import kernels_fp8 as K8
    from gguf2bin_b200.csrc.units import SHORT_WAITS
    x, w = operands(14, 512, 1024)
    rows, want, out = kernels.Fp8Rows(*held(x)), torch.empty(14, 512, device=DEV), torch.zeros(14, 512, device=DEV)
    if columns == "given":
        columns = K8.BY_THE_RULE
    fused = columns == "on the way"
    a, columns = (x, K8.WITH_X) if fused else (rows, columns)
    K8._product("test", a, w, want, K8.EPI_F32, columns=columns, split=max(split, 1))
    n = 1 << 26                                  # pairs that one block sorts: tens of milliseconds, and it lets the next kernel in at once
    idx, places, starts = torch.zeros(n, 1, dtype=torch.int32, device=DEV), torch.empty(n, dtype=torch.int32, device=DEV), torch.empty(5, dtype=torch.int32, device=DEV)
    kernels_bf16.check_status()
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    K8._product("test", a, w, out, K8.EPI_F32, columns=columns, split=max(split, 1), defines=SHORT_WAITS)
    out.zero_()
    begin.record()
    kernels.moe_sort(idx, 4, starts, places)
    K8._product("test", a, w, out, K8.EPI_F32, columns=columns, split=max(split, 1), defines=SHORT_WAITS)
    end.record()
    torch.cuda.synchronize()
    kernels_bf16.check_status()
    assert torch.equal(out, want) and begin.elapsed_time(end) > 10
