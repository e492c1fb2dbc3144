"""Routed experts in 8 bits: every instance of the experts' products, whatever the estimates would choose, and inputs that cannot be quantised on the way."""
import math

import pytest
import torch

from fp8_plain import B, EPS, blocks_of, held, matrix_values, rows_values, sum_bound
from test_gpu_fp8 import FORMS, experts_case, gated_reference
from test_gpu_kernels import DEV, rnd

pytestmark = pytest.mark.gpu


def check(x, idx, gu, down, rows, pair_row):
    """Every expert's rows against 64 bits; their places; the rows of no pair as they were (3)."""
    from gguf2bin_b200 import kernels, kernels_bf16
    kernels_bf16.check_status()
    (T, top), (E, K, I) = idx.shape, (gu.q.shape[0], gu.k, down.k)
    a, real = rows_values(*held(x)), 0
    for e in range(E):
        token, choice = torch.nonzero(idx == e, as_tuple=True)
        if not len(token):
            continue
        at = pair_row.view(T, top)[token, choice].long()
        assert torch.equal(at, torch.arange(real, real + len(token), device=DEV))
        real += len(token)
        h, bound = gated_reference(a[token], kernels.Fp8Matrix(gu.q[e], gu.scale[e], K), FORMS["silu"])
        q, s = held(h.float())
        v, m = rows_values(q, s), matrix_values(down.q[e], down.scale[e])
        # entries whose exact value is within the gate's error of a border may be one step off; a scale is off by its block's error
        steps = s.t().double().repeat_interleave(B, 1)
        want, off = (torch.nn.functional.pad(z, (0, v.shape[1] - I)) / steps for z in (h, bound))
        most = (off.view(len(token), -1, B).amax(-1) / 448).repeat_interleave(B, 1) + 4 * EPS
        step = torch.exp2(torch.floor(torch.log2(want.abs().clamp_min(2.0 ** -6))) - 3)
        to_border = (((want / step) - 0.5) - torch.round((want / step) - 0.5)).abs() * step
        moved = (to_border <= off + want.abs() * most) * step * 2
        slack = (moved * steps + v.abs() * most) @ m.abs().T
        parts = 8 * EPS                                  # the parts of K, added one after the other
        assert ((rows[at].double() - v @ m.T).abs() <= slack + (sum_bound(blocks_of(I)) * 1.2 + parts) * (v.abs() @ m.abs().T) + 1e-44).all(), e
    assert (pair_row.view(T, top)[idx >= E] == -1).all() and (rows[real:] == 3).all()


def run(x, idx, gu, down, forced=None):
    from gguf2bin_b200 import kernels_fp8 as K8
    from gguf2bin_b200.kernels import SILU
    rows, pair_row = torch.full((idx.numel(), down.q.shape[1]), 3.0, device=DEV), torch.full((idx.numel(),), 77, dtype=torch.int32, device=DEV)
    K8.moe_experts(x, idx, gu, down, rows, pair_row, SILU, None, forced)
    check(x, idx, gu, down, rows, pair_row)
    return rows, pair_row


def popular(T, top, E, seed):
    """Choices of which the first is half of the time the same expert, some have no matrices, and one expert has no row."""
    g = torch.Generator().manual_seed(seed)
    idx = torch.randint(0, E + 2, (T, top), generator=g)
    idx[torch.rand(T, generator=g) < 0.5, 0] = 1
    idx[idx == E - 2] = 0
    return idx.to(torch.int32).to(DEV)


WIDTHS = (17, 16, 32, 64, -64, 0)                        # 17: sixteen, quantised on the way; 0: the kernel of many rows
FORCED = [((c, s), (c, s)) for c in WIDTHS for s in ((1, 2, 3, 5, 8) if c else (1,))] + \
    [((a, 2), (b, 3)) for a in WIDTHS[1:5] for b in WIDTHS[1:5] if a != b] + [((16, 2), (0, 1)), ((0, 1), (16, 2)), ((-64, 1), (0, 1)), ((0, 1), (-64, 4))]


@pytest.mark.parametrize("forced", FORCED)
@pytest.mark.parametrize("T,top,E,I,K", [(7, 3, 6, 136, 640), (90, 3, 6, 264, 640), (150, 4, 40, 24, 130 * 8)])
def test_every_instance(T, top, E, I, K, forced):
    """A popular expert of several tiles, an empty one, K in one part, in several and in more than it has blocks; few pairs that the products sort."""
    x, _, _, gu, down = experts_case(T, 1, E, 0, I, K, 7)
    run(x, popular(T, top, E, T), gu, down, forced)


def test_both_products_quantise_or_neither():
    from gguf2bin_b200.kernels import KernelError
    x, _, _, gu, down = experts_case(7, 1, 6, 0, 136, 640, 7)
    for forced in (((17, 1), (16, 1)), ((16, 1), (17, 1))):
        with pytest.raises(KernelError, match="or neither"):
            run(x, popular(7, 3, 6, 1), gu, down, forced)


@pytest.mark.parametrize("T,top,E", [(1, 4, 16), (8, 4, 16), (11, 3, 5), (16, 6, 64), (300, 2, 9)])
@pytest.mark.parametrize("K,first,dtype", [(1004, 0, torch.bfloat16), (1004, 0, torch.float32), (1003, 0, torch.float32), (1003, 0, torch.bfloat16),
                                           (1000, 1, torch.bfloat16), (1000, 4, torch.bfloat16), (1000, 1, torch.float32), (1000, 2, torch.float32)])
def test_rows_that_are_quantised_first(T, top, E, K, first, dtype):
    """Widths that are no multiples of eight, and tokens that start anywhere in wider rows: on both sides of what the products sort by themselves.  The
    same rows on 16 bytes give the same bits."""
    x, _, _, gu, down = experts_case(T, 1, E, 0, 136, K, 9)
    x = rnd(T, K, seed=T).to(dtype)
    idx = popular(T, top, E, T) if E > 2 else torch.zeros(T, top, dtype=torch.int32, device=DEV)
    wide = torch.full((T, K + 13), math.nan, dtype=dtype, device=DEV)
    wide[:, first:first + K] = x
    got = run(wide[:, first:first + K], idx, gu, down)
    rows, pair_row = run(x, idx, gu, down)
    assert torch.equal(got[1], pair_row) and torch.equal(got[0], rows)
