"""The operators in 8-bit floating point against their definition: rows and matrices bit for bit, products against 64-bit sums."""
import math

import pytest
import torch

from fp8_plain import (B, EPS, F8, blocks_of, gate_up_values, held, held_matrix, matrix_values, random_matrix, rows_values, sum_bound)
from test_gpu_kernels import DEV, rnd

pytestmark = pytest.mark.gpu


def new_rows(t, k):
    from gguf2bin_b200.kernels import Fp8Rows
    return Fp8Rows(torch.full((t, blocks_of(k) * B), 77, dtype=torch.uint8, device=DEV).view(F8), torch.full((blocks_of(k), t), math.nan, device=DEV))


def same_bits(a, b):
    """Equal, NaN where NaN (of either sign)."""
    return torch.equal(a.float().nan_to_num(nan=1e9), b.float().nan_to_num(nan=1e9))


# ---- rows and matrices -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,K", [(1, 1), (1, 128), (3, 8), (17, 129), (16, 1000), (5, 1003), (129, 512), (2, 17408)])
def test_rows_are_held_as_defined(T, K, dtype):
    from gguf2bin_b200 import kernels
    x = (rnd(T, K, seed=T) * torch.logspace(-8, 8, T, device=DEV)[:, None]).to(dtype)
    x[:, K // 2] *= 300
    rows = new_rows(T, K)
    kernels.quantize_rows(x, rows)
    q, s = held(x)
    assert torch.equal(rows.q.view(torch.uint8), q.view(torch.uint8)) and torch.equal(rows.scale, s)
    # rows with a stride of their own, from an odd place on
    wide = torch.zeros(T, K + 5, dtype=dtype, device=DEV)
    wide[:, 3:3 + K] = x
    again = new_rows(T, K)
    kernels.quantize_rows(wide[:, 3:3 + K], again)
    assert torch.equal(again.q.view(torch.uint8), q.view(torch.uint8)) and torch.equal(again.scale, s)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_odd_values(dtype):
    """Zeros, the smallest and the largest values, infinities, NaN: as defined, and nothing of them in other blocks."""
    from gguf2bin_b200 import kernels
    x = rnd(12, 300, seed=1).to(dtype)
    clean = held(x)
    x[1] = 0.0
    x[2] *= 1e-38
    x[3, :128] = 2.0 ** -130
    x[4] = torch.finfo(dtype).max
    x[5, 200], x[6, 5], x[7, 299], x[8, 0] = math.inf, math.nan, -math.inf, -0.0
    rows = new_rows(12, 300)
    kernels.quantize_rows(x, rows)
    q, s = held(x)
    assert same_bits(rows.q, q) and same_bits(rows.scale, s)
    assert not rows.q[1].float().any() and rows.scale[:, 1].eq(2.0 ** -100 / torch.tensor(448.0, device=DEV)).all()
    assert rows.scale[1, 5] == math.inf and rows.scale[0, 6].isnan() and torch.equal(rows.q[5, :128].float(), clean[0][5, :128].float())
    assert rows.q[6, :128].float().isnan().all() and torch.equal(rows.q[9:].float(), clean[0][9:].float())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,K,stack", [(1, 1, 0), (128, 128, 0), (130, 257, 0), (300, 1000, 0), (24, 136, 3), (256, 128, 2)])
def test_matrices_are_held_as_defined(N, K, stack, dtype):
    from gguf2bin_b200 import kernels
    w = (rnd(max(stack, 1) * N, K, seed=N) * 0.02).to(dtype)
    m = kernels.quantize_matrix(w.view(stack, N, K) if stack else w)
    assert m.shape == ((stack, N, K) if stack else (N, K))
    for e in range(max(stack, 1)):
        q, s = held_matrix(w[e * N:(e + 1) * N])
        mine = (m.q[e], m.scale[e]) if stack else (m.q, m.scale)
        assert torch.equal(mine[0].view(torch.uint8), q.view(torch.uint8)) and torch.equal(mine[1], s)


def test_rows_go_to_their_places():
    from gguf2bin_b200 import kernels
    x = rnd(40, 200, seed=2)
    g = torch.Generator().manual_seed(1)
    at = torch.full((40, 3), -1, dtype=torch.int32)
    places = torch.randperm(130, generator=g)
    at.view(-1)[torch.randperm(120, generator=g)[:110]] = places[:110].to(torch.int32)
    rows = new_rows(130, 200)
    before = rows.q.view(torch.uint8).clone()
    kernels.quantize_rows(x, rows, at.to(DEV))
    q, s = held(x)
    token = torch.full((130,), -1)
    for t in range(40):
        for r in at[t].tolist():
            if r >= 0:
                token[r] = t
    used, unused = (token >= 0).nonzero().flatten().to(DEV), (token < 0).nonzero().flatten().to(DEV)
    src = token.to(DEV)[used]
    assert torch.equal(rows.q.view(torch.uint8)[used], q.view(torch.uint8)[src]) and torch.equal(rows.scale[:, used], s[:, src])
    assert torch.equal(rows.q.view(torch.uint8)[unused], before[unused]) and rows.scale[:, unused].isnan().all()


# ---- products --------------------------------------------------------------------------------------------------
SIZES = [(1, 64, 64), (1, 4096, 4096), (2, 300, 128), (7, 1030, 1000), (8, 640, 2048), (16, 129, 4096), (17, 256, 384), (33, 1024, 130), (64, 512, 8192),
         (65, 2048, 1024), (127, 24, 640), (128, 256, 256), (129, 257, 257), (200, 1, 1000), (256, 1536, 2048), (300, 1000, 2500), (701, 130, 7),
         (1024, 2048, 512), (2049, 384, 1100)]


def operands(M, N, K, dtype=torch.bfloat16, gated=False, stack=None):
    from gguf2bin_b200.kernels import Fp8Matrix
    x = (rnd(M, K, seed=M + 1) * torch.logspace(-3, 3, M, device=DEV)[:, None]).to(dtype)
    return x, Fp8Matrix(*random_matrix(N, K, DEV, N + K, stack, gated), K)


@pytest.mark.parametrize("M,N,K", SIZES)
def test_products(M, N, K):
    from gguf2bin_b200 import kernels, kernels_bf16
    x, w = operands(M, N, K, torch.float32 if M % 2 else torch.bfloat16)
    a, m = rows_values(*held(x)), matrix_values(w.q, w.scale)
    ref, size = a @ m.T, a.abs() @ m.abs().T
    bound = sum_bound(blocks_of(K)) * size + 1e-44
    out = torch.full((M, N), math.nan, device=DEV)
    kernels.linear(x, w, out)
    kernels_bf16.check_status()
    assert ((out.double() - ref).abs() <= bound).all()
    plain = (rows_values(*held(x)).float() @ m.float().T).double()
    assert (out.double() - ref).norm() <= max(1.5 * (plain - ref).norm(), 1e-6 * ref.norm())
    half = torch.full((M, N), math.nan, dtype=torch.bfloat16, device=DEV)
    kernels.linear(x, w, half)
    assert torch.equal(half, out.to(torch.bfloat16))
    # rows that were quantised before; an output with a stride of its own, at an odd place
    rows = kernels.Fp8Rows(*held(x))
    wide = torch.full((M, N + 5), 7.0, device=DEV)
    kernels.linear(rows, w, wide[:, 1:N + 1])
    assert torch.equal(wide[:, 1:N + 1], out) and (wide[:, 0] == 7).all() and (wide[:, N + 1:] == 7).all()
    base = rnd(M, N, seed=3)
    acc = base.clone()
    kernels.linear(rows, w, acc, accumulate=True)
    assert torch.equal(acc, base + out)
    kernels_bf16.check_status()


@pytest.mark.parametrize("M,N,K", [(1, 8, 130), (100, 257, 300), (300, 1000, 640), (530, 1537, 200)])
def test_many_rows_stored_anywhere(M, N, K):
    """The kernel of many rows, whatever the sizes would choose: outputs on 16 bytes and at odd places and strides, nothing written beside them."""
    from gguf2bin_b200 import kernels_bf16
    from gguf2bin_b200 import kernels_fp8 as K8
    from gguf2bin_b200.kernels import Fp8Rows
    x, w = operands(M, N, K)
    rows = Fp8Rows(*held(x))
    a, m = rows_values(*rows), matrix_values(w.q, w.scale)
    ref, bound = a @ m.T, sum_bound(blocks_of(K)) * (a.abs() @ m.abs().T) + 1e-44
    base, first = rnd(M, N, seed=2), None
    for before, behind in ((0, -N % 8), (1, 2), (3, 4), (8, 8 - N % 8)):
        at = slice(before, before + N)
        out, acc = torch.full((M, before + N + behind), 7.0, device=DEV), torch.full((M, before + N + behind), 7.0, device=DEV)
        half = torch.full((M, before + N + behind), 7.0, dtype=torch.bfloat16, device=DEV)
        acc[:, at] = base
        K8._product("test", rows, w, out[:, at], K8.EPI_F32, columns=0)
        K8._product("test", rows, w, acc[:, at], K8.EPI_ADD_F32, columns=0)
        K8._product("test", rows, w, half[:, at], K8.EPI_BF16, columns=0)
        kernels_bf16.check_status()
        first = out[:, at].clone() if first is None else first
        assert ((first.double() - ref).abs() <= bound).all() and torch.equal(out[:, at], first)
        assert torch.equal(acc[:, at], base + first) and torch.equal(half[:, at], first.to(torch.bfloat16))
        for t in (out, acc, half):
            assert (t[:, :before] == 7).all() and (t[:, before + N:] == 7).all()


def test_products_of_odd_rows():
    """Rows with infinities and NaN are NaN, rows of zeros zeros, and the others have the bits that they have alone."""
    from gguf2bin_b200 import kernels
    for M in (9, 150, 300):
        x, w = operands(M, 400, 300)
        clean = torch.empty(M, 400, device=DEV)
        kernels.linear(x, w, clean)
        x[1, 7], x[3, 299], x[4], x[M - 1, 128] = math.nan, math.inf, 0.0, -math.inf
        out = torch.full((M, 400), 5.0, device=DEV)
        kernels.linear(x, w, out)
        odd = [1, 3, 4, M - 1]
        rest = [i for i in range(M) if i not in odd]
        assert out[[1, 3, M - 1]].isnan().all() and not out[4].any() and torch.equal(out[rest], clean[rest])


@pytest.mark.parametrize("M", [1, 5, 40, 130, 400])
def test_matrices_side_by_side(M):
    """Matrices whose rows end inside a block of 128: each its own product, side by side."""
    from gguf2bin_b200 import kernels, kernels_fp8
    parts = [kernels.Fp8Matrix(*random_matrix(n, 200, DEV, n), 200) for n in (136, 24, 128)]
    x = rnd(M, 200, seed=4, dtype=torch.bfloat16)
    w = kernels_fp8.side_by_side(parts)
    out = torch.full((M, 288), math.nan, dtype=torch.bfloat16, device=DEV)
    kernels.linear(x, w, out)
    at = 0
    for p in parts:
        one = torch.empty(M, p.q.shape[0], dtype=torch.bfloat16, device=DEV)
        kernels.linear(x, p, one)
        assert torch.equal(out[:, at:at + p.q.shape[0]], one)
        at += p.q.shape[0]


FORMS = {"silu": (math.inf, 0.0, 1.0, 0.0), "gelu": (math.inf, 0.0, 1.5957691216057308, 0.0713548162726), "capped": (1.5, 1.0, 1.702, 0.0)}


def glu64(g, u, form):
    limit, offset, c1, c3 = form
    g, u = g.clamp_max(limit), u.clamp(-limit, limit) + offset
    return g * torch.sigmoid(g * (c1 + c3 * g * g)) * u


def gated_reference(a, w, form):
    """(value, bound of the error) of the gate in 64 bits.  The gate and the up value are off by the sums' error; the gate's slope in each is at most
    1.2 |u| (c1 and the sigmoid's slope together; 3 |u| with the capped form's c1 and GELU's cubic inside its range) and |g|; exp and the
    division are within 2^-20 of the value (fast forms)."""
    gm, um = gate_up_values(w.q, w.scale)
    g, u = a @ gm.T, a @ um.T
    c = sum_bound(a.shape[1] // B)
    dg, du = c * (a.abs() @ gm.abs().T), c * (a.abs() @ um.abs().T)
    h = glu64(g, u, form)
    return h, 3 * (u.abs() + 1 + du) * dg + (g.abs() + dg) * du + 2.0 ** -19 * (h.abs() + (g.abs() * (u.abs() + 1)) * 2.0 ** -3) + 1e-40


@pytest.mark.parametrize("name", FORMS)
@pytest.mark.parametrize("M,I,K", [(1, 8, 64), (1, 1024, 1024), (7, 136, 300), (8, 768, 2048), (17, 512, 128), (64, 384, 1000), (100, 1000, 256),
                                   (129, 128, 130), (300, 264, 1024), (1030, 640, 512)])
def test_gated_products(M, I, K, name):
    from gguf2bin_b200 import kernels, kernels_bf16
    form = FORMS[name]
    x = rnd(M, K, seed=M, dtype=torch.bfloat16)
    w = kernels.Fp8Matrix(*random_matrix(I, K, DEV, I, None, True), K)
    w = w._replace(scale=w.scale / math.sqrt(K))
    ref, bound = gated_reference(rows_values(*held(x)), w, form)
    mid = torch.full((M, I), math.nan, device=DEV)
    assert kernels.gate_up_fused(x, w, mid, 8, kernels.GluForm(*form))
    kernels_bf16.check_status()
    assert ((mid.double() - ref).abs() <= bound).all()
    # the same as quantised rows: the values' bits where the kernels that leave them are the same, else within the bound of a border
    rows = new_rows(M, I)
    assert kernels.gate_up_fused(x, w, rows, 8, kernels.GluForm(*form))
    kernels_bf16.check_status()
    check_rows(rows, ref, bound)


def check_rows(rows, ref, bound):
    """Quantised rows of values within ``bound`` of ``ref``: every scale within the bound of its block's largest value, every entry the value of an
    admissible number: rounding x (1 +- d) at the entry's own steps."""
    t, n = ref.shape
    pad = blocks_of(n) * B - n
    ref, bound = (torch.nn.functional.pad(v, (0, pad)).view(t, -1, B) for v in (ref, bound))
    scale = rows.scale.t().double()
    m = ref.abs().amax(-1).clamp_min(2.0 ** -100)
    assert ((scale * 448 - m).abs() <= bound.amax(-1) + m * 2 * EPS).all()
    got = rows.q.double().view(t, -1, B)
    want = ref / scale[..., None]
    step = torch.exp2(torch.floor(torch.log2(want.abs().clamp_min(2.0 ** -6))) - 3)         # of the binade, and of the next one up where it rounds over
    off = bound / scale[..., None] + want.abs() * 4 * EPS
    assert ((got - want).abs() <= step / 2 * (1 + 2.0 ** -30) + off * 1.1 + (want.abs() > 448) * (want.abs() - 448)).all()
    assert not got.view(t, -1)[:, n:].any()


# ---- experts ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T,top,E,identity", [(1, 1, 1, 0), (1, 4, 16, 2), (7, 3, 5, 0), (300, 2, 1024, 3), (5000, 8, 64, 0), (64, 6, 64, 0), (33, 1, 2, 6)])
def test_pairs_are_sorted_by_expert(T, top, E, identity):
    from gguf2bin_b200 import kernels
    g = torch.Generator().manual_seed(T)
    idx = torch.randint(0, E + identity, (T, top), generator=g, dtype=torch.int32)
    starts, pair_row = torch.empty(E + 1, dtype=torch.int32, device=DEV), torch.empty(T * top, dtype=torch.int32, device=DEV)
    kernels.moe_sort(idx.to(DEV), E, starts, pair_row)
    flat = idx.flatten().long()
    order = torch.argsort(flat, stable=True)
    real = int((flat < E).sum())
    want = torch.full((T * top,), -1, dtype=torch.int32)
    want[order[:real]] = torch.arange(real, dtype=torch.int32)
    assert torch.equal(pair_row.cpu(), want)
    assert torch.equal(starts.cpu().long(), torch.searchsorted(flat[order].contiguous(), torch.arange(E + 1)))


def experts_case(T, top, E, identity, I, K, seed, hot=0.0):
    from gguf2bin_b200.kernels import Fp8Matrix
    g = torch.Generator().manual_seed(seed)
    n = E + identity
    p = torch.ones(n) + hot * torch.tensor([1.0] + [0.0] * (n - 1)) * n
    idx = torch.multinomial(p.expand(T, n), top, generator=g).to(torch.int32).to(DEV)
    weight = torch.rand(T, top, generator=g).to(DEV)
    gu = Fp8Matrix(*random_matrix(I, K, DEV, seed, E, True), K)
    gu = gu._replace(scale=gu.scale / math.sqrt(K))
    return rnd(T, K, seed=seed, dtype=torch.bfloat16), idx, weight, gu, Fp8Matrix(*random_matrix(K, I, DEV, seed + 1, E), I)


# one token; fewer rows than experts; a hot expert with several tiles; empty experts; every choice without matrices possible
@pytest.mark.parametrize("T,top,E,identity,I,K,hot", [(1, 1, 1, 0, 8, 64, 0), (1, 4, 16, 2, 768, 512, 0), (16, 6, 64, 0, 136, 256, 1), (33, 2, 7, 1, 96, 1000, 0),
                                                      (200, 3, 8, 0, 200, 384, 3), (700, 4, 12, 2, 384, 512, 2), (1500, 2, 3, 5, 128, 136, 0)])
def test_experts(T, top, E, identity, I, K, hot):
    from gguf2bin_b200 import kernels, kernels_bf16
    x, idx, weight, gu, down = experts_case(T, top, E, identity, I, K, 11, hot)
    rows, pair_row = torch.full((T * top, K), 3.0, device=DEV), torch.empty(T * top, dtype=torch.int32, device=DEV)
    kernels.moe_experts_fp8(x, idx, gu, down, rows, pair_row)
    kernels_bf16.check_status()
    a = rows_values(*held(x))
    real = 0
    y = torch.zeros(T, K, dtype=torch.float64, device=DEV)
    for e in range(E + identity):
        token, choice = torch.nonzero(idx == e, as_tuple=True)
        if not len(token):
            continue
        at = pair_row.view(T, top)[token, choice].long()
        if e >= E:
            assert (at == -1).all()
            y.index_add_(0, token, x[token].double() * weight[token, choice].double()[:, None])
            continue
        assert torch.equal(at, torch.arange(real, real + len(token), device=DEV))
        real += len(token)
        h, bound = gated_reference(a[token], kernels.Fp8Matrix(gu.q[e], gu.scale[e], K), FORMS["silu"])
        q, s = held(h.float())
        v, m = rows_values(q, s), matrix_values(down.q[e], down.scale[e])
        ref = v @ m.T
        # entries whose exact value is within the gate's error of a border may be one step off; a scale is off by its block's error
        steps = s.t().double().repeat_interleave(B, 1)
        pad = torch.nn.functional.pad
        want, off = pad(h, (0, v.shape[1] - I)) / steps, pad(bound, (0, v.shape[1] - I)) / steps
        most = (off.view(len(token), -1, B).amax(-1) / 448).repeat_interleave(B, 1) + 4 * EPS           # relative change of the block's scale
        step = torch.exp2(torch.floor(torch.log2(want.abs().clamp_min(2.0 ** -6))) - 3)
        to_border = (((want / step) - 0.5) - torch.round((want / step) - 0.5)).abs() * step
        moved = (to_border <= off + want.abs() * most) * step * 2
        slack = (moved * steps + v.abs() * most) @ m.abs().T
        assert ((rows[at].double() - ref).abs() <= slack + sum_bound(blocks_of(I)) * (v.abs() @ m.abs().T) * 1.2 + 1e-44).all()
        y.index_add_(0, token, rows[at].double() * weight[token, choice].double()[:, None])
    assert (rows[real:] == 3).all()
    for dtype, eps in ((torch.float32, 0), (torch.bfloat16, 2.0 ** -8)):
        out = torch.full((T, K), math.nan, dtype=dtype, device=DEV)
        kernels.moe_back(rows, pair_row, weight, x, out)
        spread = sum((weight[:, j:j + 1].double() * torch.where(pair_row.view(T, top)[:, j:j + 1] >= 0, rows[pair_row.view(T, top)[:, j].clamp_min(0).long()].double(),
                                                                  x.double())).abs() for j in range(top))
        assert ((out.double() - y).abs() <= eps * y.abs() + (top + 1) * EPS * spread * (1 + eps) + 1e-40).all()
    base = rnd(T, K, seed=6)
    acc, out = base.clone(), torch.empty(T, K, device=DEV)
    kernels.moe_back(rows, pair_row, weight, x.float(), out)
    kernels.moe_back(rows, pair_row, weight, x.float(), acc, accumulate=True)
    assert torch.equal(acc, base + out)


@pytest.mark.parametrize("T,top,E,what", [(32, 1, 3, "one"), (11, 3, 5, "one"), (128, 1, 3, "one"), (16, 2, 1024, "spread"), (64, 2, 1024, "spread"),
                                          (33, 4, 200, "spread"), (10, 3, 7, "twice"), (40, 3, 7, "twice"), (300, 3, 7, "twice"), (9, 2, 6, "nobody"),
                                          (40, 2, 6, "nobody"), (400, 2, 6, "nobody"), (5, 6, 9, "outside"), (21, 6, 9, "outside"), (150, 6, 9, "outside")])
def test_choices_of_every_kind(T, top, E, what):
    """Few pairs, which the products sort by themselves, on both sides of their limit, and many: all of one expert, each of another, the same expert
    twice in a token, numbers that no expert has.  Every row against the one that its expert alone gives its token."""
    from gguf2bin_b200 import kernels, kernels_bf16
    K, I = 256, 136
    g = torch.Generator().manual_seed(T)
    idx = {"one": torch.full((T, top), E - 1), "spread": torch.randint(0, E, (T, top), generator=g), "nobody": torch.full((T, top), E),
           "twice": torch.randint(0, E, (T, 1), generator=g).expand(T, top),
           "outside": torch.randint(-3, E + 3, (T, top), generator=g)}[what].to(torch.int32).contiguous().to(DEV)
    x, _, weight, gu, down = experts_case(T, 1, E, 0, I, K, 3)
    rows, pair_row = torch.full((T * top, K), 3.0, device=DEV), torch.full((T * top,), 77, dtype=torch.int32, device=DEV)
    kernels.moe_experts_fp8(x, idx, gu, down, rows, pair_row)
    kernels_bf16.check_status()
    flat = idx.flatten().long()
    real = (flat >= 0) & (flat < E)
    order = torch.argsort(torch.where(real, flat, E), stable=True)[:int(real.sum())]
    want = torch.full_like(pair_row, -1)
    want[order] = torch.arange(len(order), dtype=torch.int32, device=DEV)
    assert torch.equal(pair_row, want) and (rows[len(order):] == 3).all()
    for e in flat[order].unique().tolist():
        pairs = order[flat[order] == e]
        one = torch.full((len(pairs), K), math.nan, device=DEV)
        kernels.moe_experts_fp8(x[pairs // top].contiguous(), torch.zeros(len(pairs), 1, dtype=torch.int32, device=DEV),
                                kernels.Fp8Matrix(gu.q[e:e + 1], gu.scale[e:e + 1], K), kernels.Fp8Matrix(down.q[e:e + 1], down.scale[e:e + 1], I), one,
                                torch.empty(len(pairs), dtype=torch.int32, device=DEV))
        got = rows[pair_row[pairs].long()]
        # sums of K in other parts may move a value between over a border of e4m3: by a step, 2^-3 of it at most, were it all of them.  Another row's
        # or expert's values are off by 2^0.5
        assert (got - one).norm() <= 2.0 ** -3 * one.norm()
    kernels_bf16.check_status()


def test_a_feed_forward_on_another_stream_and_in_graphs():
    """Norm-sized rows -> gated product -> rows -> down product added to a stream: on a side stream, captured twice over one workspace, replayed in
    turn with new inputs; the bits of plain calls."""
    from gguf2bin_b200 import kernels
    from gguf2bin_b200.engine.workspace import Workspace
    K, I = 640, 392
    gu, down = kernels.Fp8Matrix(*random_matrix(I, K, DEV, 1, None, True), K), kernels.Fp8Matrix(*random_matrix(K, I, DEV, 2), I)

    def step(x, y, ws):
        rows = kernels.Fp8Rows(ws.buffer("mid.q", (len(x), 512), F8), ws.buffer("mid.s", (4, len(x)), torch.float32))
        kernels.gate_up_fused(x, gu, rows, 8, workspace=ws)
        kernels.linear(rows, down, y, accumulate=True, workspace=ws)

    inputs = [rnd(T, K, seed=T, dtype=torch.bfloat16) for T in (3, 150)]
    want = []
    for x in inputs:
        y = torch.ones(len(x), K, device=DEV)
        step(x, y, Workspace(DEV))
        want.append(y)
    torch.cuda.synchronize()
    ws, side = Workspace(DEV), torch.cuda.Stream()
    outs, graphs = [torch.empty_like(y) for y in want], []
    with torch.cuda.stream(side):
        for _ in range(2):
            for x, y in zip(inputs, outs):
                y.fill_(1)
                step(x, y, ws)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    bufs = [torch.zeros_like(x) for x in inputs]
    for x, y in zip(bufs, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y.fill_(1)
            step(x, y, ws)
        graphs.append(g)
    for x, b in zip(inputs, bufs):
        b.copy_(x)
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_the_first_product_is_not_captured(monkeypatch):
    """The word that waits report to would be the graph's own memory: refused, and a later capture is what a call is."""
    from gguf2bin_b200 import kernels, kernels_bf16
    from gguf2bin_b200 import kernels_fp8 as K8
    x, w = operands(20, 64, 256)
    want, out = torch.empty(20, 64, device=DEV), torch.empty(20, 64, device=DEV)
    kernels.linear(x, w, want)
    word = dict(kernels_bf16._status)
    K8._plans.clear()
    kernels_bf16._status.clear()
    try:
        with pytest.raises(kernels.KernelError, match="captured"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                kernels.linear(x, w, out)
    finally:
        kernels_bf16._status.update(word)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kernels.linear(x, w, out)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    kernels_bf16.check_status()


def test_two_streams_at_once():
    """Products of every kernel and experts on two streams at the same time, without a workspace: each call has scratch memory of its own."""
    from gguf2bin_b200 import kernels, kernels_bf16
    cases = [operands(M, 512, 1000) for M in (3, 40, 200, 1500)]
    h, idx, _, gu, down = experts_case(70, 3, 9, 0, 136, 256, 5)

    def run():
        outs = [torch.empty(len(x), 512, device=DEV) for x, _ in cases]
        for (x, w), y in zip(cases, outs):
            kernels.linear(x, w, y)
        outs.append(torch.zeros(210, 256, device=DEV))
        kernels.moe_experts_fp8(h, idx, gu, down, outs[-1], torch.empty(210, dtype=torch.int32, device=DEV))
        return outs

    want = run()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(run())
    torch.cuda.synchronize()
    kernels_bf16.check_status()
    assert all(torch.equal(a, b) for outs in got for a, b in zip(outs, want))


def test_empty_and_repeated_calls():
    from gguf2bin_b200 import kernels
    x, w = operands(0, 64, 64)
    kernels.linear(x, w, torch.empty(0, 64, device=DEV))
    kernels.gate_up_fused(x, kernels.Fp8Matrix(*random_matrix(64, 64, DEV, 1, None, True), 64), torch.empty(0, 64, device=DEV), 8)
    x, w = operands(50, 300, 700)
    outs = [torch.empty(50, 300, device=DEV) for _ in range(4)]
    for o in outs:
        kernels.linear(x, w, o)
    assert all(torch.equal(o, outs[0]) for o in outs)


@pytest.mark.parametrize("kernel", ["tc store", "tc rows", "few", "few parts", "on the way"])
def test_products_whose_copies_never_come(kernel):
    """The build whose copy role issues nothing: every wait runs out, the kernel returns and the host learns of it."""
    from gguf2bin_b200 import kernels, kernels_bf16
    from gguf2bin_b200 import kernels_fp8 as K8
    from gguf2bin_b200.csrc.units import WAITS_RUN_OUT
    kernels_bf16.check_status()
    M = 300 if kernel.startswith("tc") else 20
    x, w = operands(M, 512, 1024)
    rows, out = kernels.Fp8Rows(*held(x)), torch.zeros(M, 512, device=DEV)
    if kernel == "tc rows":
        gated = kernels.Fp8Matrix(*random_matrix(256, 1024, DEV, 1, None, True), 1024)
        K8._product("test", rows, gated, new_rows(M, 256), K8.EPI_GATED_ROWS, columns=0, defines=WAITS_RUN_OUT)
    else:
        columns, split = {"tc store": (0, 1), "few": (32, 1), "few parts": (32, 4), "on the way": (K8.WITH_X, 2)}[kernel]
        K8._product("test", x if kernel == "on the way" else rows, w, out, K8.EPI_F32, columns=columns, split=split, defines=WAITS_RUN_OUT)
    torch.cuda.synchronize()
    with pytest.raises(kernels.KernelError, match="gemm_fp8.*gave up waiting"):
        kernels_bf16.check_status()
    kernels.linear(rows, w, out)
    kernels_bf16.check_status()
    again = torch.empty_like(out)
    kernels.linear(x, w, again)
    assert torch.equal(out, again) and out.abs().sum() > 0


FEW = [(M, N, K, columns, split) for M, N, K in ((1, 130, 300), (13, 128, 1024), (40, 300, 2176), (150, 200, 640), (5, 64, 5000), (17, 72, 200))
       for columns in ("on the way", 16, 32, 64, -64) for split in (1, 2, 3, 4, 7, 8)
       if K % 8 == 0 or columns != "on the way"]         # (rows of other lengths are quantised first)


@pytest.mark.parametrize("M,N,K,columns,split", FEW)
def test_every_shape_of_few_rows(M, N, K, columns, split):
    """Each width and number of parts, ranges of K that are empty or of several chunks of scales, several tiles of rows."""
    from gguf2bin_b200 import kernels, kernels_bf16
    from gguf2bin_b200 import kernels_fp8 as K8
    x, w = operands(M, N, K)
    rows = kernels.Fp8Rows(*held(x))
    a, m = rows_values(*rows), matrix_values(w.q, w.scale)
    out = torch.full((M, N), math.nan, device=DEV)
    fused = columns == "on the way"
    K8._product("test", x if fused else rows, w, out, K8.EPI_F32, columns=K8.WITH_X if fused else columns, split=split)
    kernels_bf16.check_status()
    assert ((out.double() - a @ m.T).abs() <= (sum_bound(blocks_of(K)) + 8 * EPS) * (a.abs() @ m.abs().T) + 1e-44).all()
    g = kernels.Fp8Matrix(*random_matrix(N // 16 * 8, K, DEV, 5, None, True), K)
    g = g._replace(scale=g.scale / math.sqrt(K))
    x = rnd(M, K, seed=M, dtype=torch.bfloat16)
    ref, bound = gated_reference(rows_values(*held(x)), g, FORMS["silu"])
    mid = torch.full((M, N // 16 * 8), math.nan, device=DEV)
    x = x.float() if M % 2 else x
    K8._product("test", x if fused else kernels.Fp8Rows(*held(x)), g, mid, K8.EPI_GATED_F32, columns=K8.WITH_X if fused else columns, split=split)
    kernels_bf16.check_status()
    assert ((mid.double() - ref).abs() <= bound).all()
