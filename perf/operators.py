"""The operators of 8-bit floating point (e4m3, a scale for each block of 128) as cases that can be timed and checked.

* ``op`` "rows": activations quantised, a scale per row and 128 columns.
* ``op`` "product": activations times a matrix in 8 bits whose scales belong to blocks of 128 x 128; the product is stored in
  bfloat16 or float32, or added to a float32 stream.
* ``op`` "gated": the same with a gate and an up matrix and silu(gate) * up behind them, left as float32 or as quantised rows
  for the product that follows.
* ``op`` "experts": tokens sorted by the experts that were chosen for them, the experts' gated and down products, and the results
  brought back to the tokens with the choices' weights applied.

A block x of 128 values is held as m = max(max |x|, 2^-100), scale m / 448 and e4m3(x * (448 / m)), every step one operation in
32 bits.  A gate/up matrix is one matrix whose rows alternate, eight gate rows and then the eight up rows of the same outputs.
"""
from __future__ import annotations

import math

import torch

own = False

B, MOST, TINY = 128, 448.0, 2.0 ** -100


# ---- the cases -------------------------------------------------------------------------------------------------
def listed():
    return [
        # the input of a product for one token of a decode step: latency
        dict(name="rows_one", op="rows", tokens=1, k=4096, dtype="float32"),
        # a batch of long prompts in front of a layer's first product
        dict(name="rows_prompt", op="rows", tokens=8192, k=4096, dtype="bfloat16"),
        # one user's decode step: q, k and v of an 8B model's layer
        dict(name="product_one", op="product", tokens=1, n=6144, k=4096, dtype="bfloat16", out="bfloat16"),
        # 64 sequences: the down product of a 14B model's feed-forward, added to the stream
        dict(name="product_batch", op="product", tokens=64, n=5120, k=17408, dtype="float32", out="stream"),
        # sizes that are multiples of nothing
        dict(name="product_odd", op="product", tokens=701, n=1030, k=2500, dtype="bfloat16", out="float32"),
        # a prompt of 2,048 tokens: q, k and v of an 8B model's layer
        dict(name="product_prompt", op="product", tokens=2048, n=6144, k=4096, dtype="bfloat16", out="bfloat16"),
        # eight prompts of 1,024 tokens: the down product of an 8B model, added to the stream
        dict(name="product_long", op="product", tokens=8192, n=4096, k=12288, dtype="bfloat16", out="stream"),
        # eight sequences: gate and up of an 8B model's feed-forward
        dict(name="gated_batch", op="gated", tokens=8, inter=12288, k=4096, dtype="bfloat16", out="float32"),
        # a prompt: gate and up of a 14B model's feed-forward, left as the rows that the down product reads
        dict(name="gated_prompt", op="gated", tokens=2048, inter=17408, k=5120, dtype="bfloat16", out="rows"),
        # one sequence through a routed layer
        dict(name="experts_one", op="experts", tokens=1, experts=16, identity=2, top=4, inter=768, k=2048, skew=0.0),
        # sixteen sequences, more experts than rows for each
        dict(name="experts_batch", op="experts", tokens=16, experts=64, identity=0, top=6, inter=768, k=2048, skew=1.0),
        # long prompts through a routed layer, some experts far more popular than others
        dict(name="experts_prompt", op="experts", tokens=4096, experts=32, identity=0, top=4, inter=1536, k=2048, skew=0.5),
    ]


def draw(rng):
    def log_int(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    def size(lo, hi, step):                      # half of them multiples of a block, half of anything that the operator takes
        n = log_int(lo, hi)
        return max(B, n // B * B) if rng.random() < 0.5 else max(step, n // step * step)

    op = rng.choice(["rows", "product", "product", "product", "gated", "gated", "experts", "experts"])
    if op == "rows":
        k = size(64, 17408, 1)
        return dict(op=op, tokens=log_int(1, min(8192, 50_000_000 // k)), k=k, dtype=rng.choice(["bfloat16", "float32"]))
    if op == "product":
        n, k = size(64, 17408, 1), size(64, 17408, 1)
        return dict(op=op, tokens=log_int(1, min(8192, 400_000_000_000 // (n * k))), n=n, k=k, dtype=rng.choice(["bfloat16", "float32"]),
                    out=rng.choice(["bfloat16", "float32", "stream"]))
    if op == "gated":
        inter, k = size(64, 17408, 8), size(64, 8192, 1)
        return dict(op=op, tokens=log_int(1, min(4096, 200_000_000_000 // (inter * k))), inter=inter, k=k,
                    dtype=rng.choice(["bfloat16", "float32"]), out=rng.choice(["float32", "rows"]))
    experts, identity = log_int(1, 64), rng.choice([0, 0, 0, 2])
    top = rng.randint(1, min(8, experts + identity))
    return dict(op=op, tokens=log_int(1, 4096), experts=experts, identity=identity, top=top, inter=size(64, 1536, 8), k=size(64, 2048, 8),
                skew=rng.choice([0.0, 0.5, 1.0, 2.0]))


def _blocks(n):
    return -(-n // B)


# ---- inputs ----------------------------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _activations(rows, k, dtype, g):
    """Normal entries; a few channels far larger than the others, and rows of unequal size, as hidden states are."""
    x = torch.randn(rows, k, device="cuda", generator=g)
    x *= torch.exp(1.5 * torch.randn(rows, 1, device="cuda", generator=g))
    x *= torch.where(torch.rand(k, device="cuda", generator=g) < 0.01, 20.0, 1.0)
    return x.to(dtype)


def _matrix(n, k, g, count=None):
    """An e4m3 matrix, rows filled up with zeros to whole blocks, and the scales of its blocks."""
    kb, nb, lead = _blocks(k), _blocks(n), () if count is None else (count,)
    q = torch.empty(*lead, n, kb * B, dtype=torch.float8_e4m3fn, device="cuda")
    for e in q.unsqueeze(0) if count is None else q:           # one at a time: the values are four times as large
        v = torch.randn(n, kb * B, device="cuda", generator=g).mul_(120.0).clamp_(-MOST, MOST)
        v[:, k:] = 0.0
        e.copy_(v)
    scale = 0.02 / 120.0 * torch.exp(0.3 * torch.randn(*lead, nb, kb, device="cuda", generator=g))
    return q, scale


def _gate_up(inter, k, g, count=None):
    """Gate and up rows in eights in turn, and both matrices' scales side by side."""
    q, _ = _matrix(2 * inter, k, g, count)
    lead = () if count is None else (count,)
    return q, 0.02 / 120.0 * torch.exp(0.3 * torch.randn(*lead, 2, _blocks(inter), _blocks(k), device="cuda", generator=g))


def prepare(case, seed):
    g = _generator(seed)
    s = dict(case)
    if case["op"] == "experts":
        t, e, n, top = case["tokens"], case["experts"], case["identity"], case["top"]
        s["x"] = _activations(t, case["k"], torch.bfloat16, g)
        popular = -case["skew"] * torch.log(torch.arange(1, e + n + 1, device="cuda", dtype=torch.float32))
        noise = -torch.log(-torch.log(torch.rand(t, e + n, device="cuda", generator=g).clamp_(1e-9, 1 - 1e-7)))
        score, idx = torch.topk(popular + noise, top, dim=1)
        s["idx"], s["weight"] = idx.to(torch.int32).contiguous(), torch.softmax(score, dim=1).contiguous()
        s["most"] = max(1, int(torch.bincount(idx.flatten(), minlength=e + n)[:e].max()))     # for the plain form's padded ranges
        s["wq"], s["ws"] = _gate_up(case["inter"], case["k"], g, e)
        s["dq"], s["ds"] = _matrix(case["k"], case["inter"], g, e)
        return s
    s["x"] = _activations(case["tokens"], case["k"], getattr(torch, case["dtype"]), g)
    if case["op"] == "product":
        s["wq"], s["ws"] = _matrix(case["n"], case["k"], g)
        if case["out"] == "stream":
            s["stream"] = torch.randn(case["tokens"], case["n"], device="cuda", generator=g)
    elif case["op"] == "gated":
        s["wq"], s["ws"] = _gate_up(case["inter"], case["k"], g)
    return s


# ---- the plain form --------------------------------------------------------------------------------------------
def _quantised(x):
    """(q [rows, blocks, 128], scale [rows, blocks]) of float32 ``x`` [..., K]; q in e4m3."""
    k = x.shape[-1]
    x = torch.nn.functional.pad(x, (0, _blocks(k) * B - k)).unflatten(-1, (-1, B))
    m = x.abs().amax(-1).clamp_min(TINY)
    most = torch.full_like(m, MOST)              # (a division by a number would be a product with its reciprocal)
    return (x * (most / m)[..., None]).to(torch.float8_e4m3fn), m / most


def _values(x):
    """What quantised rows of ``x`` stand for, without their scales' rounding."""
    q, scale = _quantised(x.float())
    return (q.float() * scale[..., None]).flatten(-2)


def _matrix_values(q, scale):
    """Float32 values of a matrix (or a stack) from its entries and its blocks' scales."""
    n = q.shape[-2]
    rows = scale.repeat_interleave(B, dim=-2)[..., :n, :]
    return (q.float().unflatten(-1, (-1, B)) * rows[..., None]).flatten(-2)


def _gate_up_values(q, scale):
    """The same for gate and up apart."""
    both = q.unflatten(-2, (-1, 2, 8))
    return (_matrix_values(both.select(-3, i).flatten(-3, -2), scale.select(-3, i)) for i in (0, 1))


def _silu(z):
    return z / (1.0 + torch.exp(-z))


def _experts_plain(s):
    t, top, e, most = s["tokens"], s["top"], s["experts"], s["most"]
    x = s["x"].float()
    pair = s["idx"].flatten().long()
    order = torch.argsort(pair, stable=True)
    counts = (pair[:, None] == torch.arange(e, device="cuda")).sum(0)
    first = torch.cumsum(counts, 0) - counts
    place = torch.arange(most, device="cuda")
    used = place < counts[:, None]                                                    # [experts, most]
    at = order[(first[:, None] + place).clamp_max(t * top - 1)]                       # the pair in each place
    rows = _values(x)[at // top]
    gate, up = _gate_up_values(s["wq"], s["ws"])
    h = _silu(rows @ gate.transpose(1, 2)) * (rows @ up.transpose(1, 2))
    y = _values(h) @ _matrix_values(s["dq"], s["ds"]).transpose(1, 2)
    back = x.repeat_interleave(top, dim=0)                                            # an expert without matrices returns its input
    back[at[used]] = y[used]
    return (back.view(t, top, -1) * s["weight"][..., None]).sum(1).to(torch.bfloat16)


def _plain(s):
    if s["op"] == "experts":
        return _experts_plain(s)
    if s["op"] == "rows":
        q, scale = _quantised(s["x"].float())
        return q.flatten(-2), scale.t().contiguous()
    x = _values(s["x"])
    if s["op"] == "product":
        y = x @ _matrix_values(s["wq"], s["ws"]).t()
        if s["out"] == "stream":
            return s["stream"].add_(y)
        return y.to(getattr(torch, s["out"]))
    gate, up = _gate_up_values(s["wq"], s["ws"])
    h = _silu(x @ gate.t()) * (x @ up.t())
    if s["out"] == "float32":
        return h
    q, scale = _quantised(h)
    return q.flatten(-2), scale.t().contiguous()


# ---- the framework's calls -------------------------------------------------------------------------------------
def _rows_for(kernels, tokens, k):
    return kernels.Fp8Rows(torch.empty(tokens, _blocks(k) * B, dtype=torch.float8_e4m3fn, device="cuda"),
                           torch.empty(_blocks(k), tokens, device="cuda"))


def _own(s):
    from gguf2bin_b200 import kernels
    t, x = s["tokens"], s["x"]
    if s["op"] == "rows":
        rows = _rows_for(kernels, t, s["k"])
        kernels.quantize_rows(x, rows)
        return rows.q, rows.scale
    w = kernels.Fp8Matrix(s["wq"], s["ws"], s["k"])
    if s["op"] == "product":
        if s["out"] == "stream":
            kernels.linear(x, w, s["stream"], accumulate=True)
            return s["stream"]
        y = torch.empty(t, s["n"], dtype=getattr(torch, s["out"]), device="cuda")
        kernels.linear(x, w, y)
        return y
    if s["op"] == "gated":
        if s["out"] == "rows":
            rows = _rows_for(kernels, t, s["inter"])
            kernels.gate_up_fused(x, w, rows, 8)
            return rows.q, rows.scale
        h = torch.empty(t, s["inter"], device="cuda")
        kernels.gate_up_fused(x, w, h, 8)
        return h
    rows = torch.empty(t * s["top"], s["k"], device="cuda")
    pair_row = torch.empty(t * s["top"], dtype=torch.int32, device="cuda")
    kernels.moe_experts_fp8(x, s["idx"], w, kernels.Fp8Matrix(s["dq"], s["ds"], s["inter"]), rows, pair_row)
    out = torch.empty(t, s["k"], dtype=torch.bfloat16, device="cuda")
    kernels.moe_back(rows, pair_row, s["weight"], x, out)
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------
def work(case):
    t, k = case["tokens"], case["k"]
    size = 4 if case.get("dtype") == "float32" else 2
    if case["op"] == "rows":
        return {"bytes": t * k * (size + 1) + 4 * t * _blocks(k), "flops": 3 * t * k}
    if case["op"] == "product":
        n = case["n"]
        out = {"bfloat16": 2, "float32": 4, "stream": 8}[case["out"]]
        return {"bytes": t * k * size + n * k + 4 * _blocks(n) * _blocks(k) + t * n * out, "flops": 2 * t * n * k}
    if case["op"] == "gated":
        i = case["inter"]
        out = 4 * t * i if case["out"] == "float32" else t * i + 4 * t * _blocks(i)
        return {"bytes": t * k * size + 2 * i * k + 8 * _blocks(i) * _blocks(k) + out, "flops": 4 * t * i * k}
    e, top, i = case["experts"], case["top"], case["inter"]
    real = e / (e + case["identity"])                                      # the share of the choices that are experts with matrices
    pairs = t * top * real
    used = e * (1.0 - (1.0 - min(1.0, top / (e + case["identity"]))) ** t) if case["skew"] == 0 else min(e, pairs)
    return {"bytes": used * 3 * i * k + 4 * t * k + 8 * t * top, "flops": 6 * pairs * i * k}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------
def _rounded(v):
    """e4m3 nearest to each of ``v`` (float64), ties to even: three bits behind the first, exponents from -6 on."""
    exponent = torch.frexp(v).exponent.double() - 1.0
    step = torch.exp2(exponent.clamp_min(-6.0) - 3.0)
    return (torch.round(v / step) * step).clamp(-MOST, MOST)


def _held(x):
    """(values in 64 bits, scales in 64 bits) of the rows that 32-bit ``x`` is held as."""
    t, k = x.shape
    full = torch.zeros(t, _blocks(k) * B, dtype=torch.float32, device=x.device)
    full[:, :k] = x
    blocks = full.view(t, -1, B)
    m = torch.maximum(blocks.max(-1).values, -blocks.min(-1).values).double().clamp_min(TINY)
    inverse = (MOST / m).float()                 # one rounding of the exact quotient: 64 bits hold more than twice 32's
    return _rounded((blocks * inverse[..., None]).double()), m / MOST


def _double_matrix(q, scale):
    n, padded = q.shape
    v = q.to(torch.float64).view(n, padded // B, B)
    at = torch.arange(n, device=q.device) // B
    return (v * scale.to(torch.float64)[at][:, :, None]).view(n, padded)


def _double_rows(x):
    v, scale = _held(x)
    return (v * scale.float().double()[..., None]).flatten(1)


def _double_gated(x, q, scale):
    inter = q.shape[0] // 2
    at = torch.arange(inter, device=q.device)
    gate_rows = at // 8 * 16 + at % 8
    g = x @ _double_matrix(q[gate_rows], scale[0]).t()
    return g * torch.sigmoid(g) * (x @ _double_matrix(q[gate_rows + 8], scale[1]).t())


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rows":
        v, scale = _held(s["x"].float())
        return v.flatten(1), scale.t().contiguous()
    x = _double_rows(s["x"].float())
    if case["op"] == "product":
        y = x @ _double_matrix(s["wq"], s["ws"]).t()
        return y + s["stream"].double() if case["out"] == "stream" else y
    if case["op"] == "gated":
        h = _double_gated(x, s["wq"], s["ws"])
        if case["out"] == "float32":
            return h
        v, scale = _held(h.float())
        return v.flatten(1), scale.t().contiguous()
    t, top = case["tokens"], case["top"]
    out = torch.zeros(t, case["k"], dtype=torch.float64, device="cuda")
    weight, idx = s["weight"].double(), s["idx"].long()
    for e in range(case["experts"] + case["identity"]):
        token, choice = torch.nonzero(idx == e, as_tuple=True)
        if not len(token):
            continue
        if e < case["experts"]:
            h = _double_gated(x[token], s["wq"][e], s["ws"][e])
            y = _double_rows(h.float()) @ _double_matrix(s["dq"][e], s["ds"][e]).t()
        else:
            y = s["x"][token].double()
        out.index_add_(0, token, y * weight[token, choice][:, None])
    return out
