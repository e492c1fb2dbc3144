"""Bindings of the kernels in 8-bit floating point (``csrc/fp8.cuh`` says how values are held)."""
from __future__ import annotations

from ctypes import Structure, addressof, c_float, c_int, c_longlong, c_void_p
from typing import Optional

import torch

from . import kernels
from .kernels_bf16 import _status, _status_word
from .kernels import SILU, Fp8Matrices, Fp8Matrix, Fp8Rows, KernelError, _call, _code, _fn, _ptr, _stream

ON_THE_WAY = 16                      # rows up to which a product may quantise them itself (whether it does: choose in csrc/products_fp8.cu)
BLOCK = 128                          # values of a row, and of either side of a matrix, that share a scale
F8 = torch.float8_e4m3fn
MOST_EXPERTS = 1024                  # csrc/fp8.cuh
SORTED_AT_ONCE = 32 * 32 * 8         # pairs that the sort's block walks on by (csrc/quant_fp8.cuh)
EPI_BF16, EPI_F32, EPI_ADD_F32, EPI_GATED_F32, EPI_GATED_ROWS = 0, 1, 2, 3, 4


def blocks_of(n: int) -> int:
    return -(-n // BLOCK)


def new_rows(tokens: int, k: int, workspace, name: str, device) -> Fp8Rows:
    """Room for the quantised rows of ``tokens`` times ``k`` values: of the workspace, or, without one, new."""
    kb = blocks_of(k)
    if workspace is None:
        return Fp8Rows(torch.empty((tokens, kb * BLOCK), dtype=F8, device=device),
                       torch.empty((kb, tokens), dtype=torch.float32, device=device))
    return Fp8Rows(workspace.buffer(name + ".q", (tokens, kb * BLOCK), F8), workspace.buffer(name + ".scale", (kb, tokens), torch.float32))


class _Call(Structure):
    """What a call's sizes and types fix (csrc/products_fp8.cu)."""
    _fields_ = [(n, c_longlong) for n in ("lda", "lds", "ldw", "ldo", "ldos", "x_stride")] + \
        [(n, c_int) for n in ("M", "N", "K", "x_dtype", "epi", "n_experts", "top", "H", "columns", "split", "with_x", "columns_2", "split_2", "with_x_2")] + \
        [(n, c_float) for n in ("limit", "offset", "c1", "c3")]


class _Plan:
    """A call that was checked once: every later one of the same sizes, strides, types, alignments and devices only passes its addresses."""
    __slots__ = ("call", "at", "scratch", "status", "f")


_plans: dict = {}
BY_THE_RULE, WITH_X = 1, 17          # in place of columns 16, 32, 64, -64 (gemm_fp8_few.cuh) and 0 (gemm_fp8_tc.cuh); WITH_X: 16, quantised on the way


def _f(name: str, argtypes, defines=()):
    return _fn("products_fp8.cu", name, argtypes, defines=tuple(defines))


def _plan(key, call: _Call, device, prepare: str, name: str, argtypes, x_aligned: bool, by_rule: bool = True, defines=()) -> _Plan:
    if device not in _status and torch.cuda.is_current_stream_capturing():
        # (the word that waits report to would be the graph's own memory, and gone with it)
        raise KernelError(f"{name[4:]}: the first product on {device} cannot be captured; run it once before")
    plan = _Plan()
    plan.call, plan.at = call, addressof(call)
    size = _f(prepare, [c_void_p, c_int, c_int], defines)
    size.restype = c_longlong
    plan.scratch = size(plan.at, 1 if x_aligned else 0, 1 if by_rule else 0)
    plan.status = _status_word(device).data_ptr()
    plan.f = _f(name, argtypes, defines)
    if len(_plans) > 4096:
        _plans.clear()
    _plans[key] = plan
    return plan


def _failed(f) -> None:
    raise KernelError(f._lib.g2b_last_error().decode("utf-8", "replace"))


def _scratch(plan: _Plan, workspace, name: str, device):
    if workspace is not None:
        workspace.waits = True
        return workspace.buffer(name, (plan.scratch,), torch.uint8).data_ptr() if plan.scratch else None, None
    if not plan.scratch:
        return None, None
    buf = torch.empty(plan.scratch, dtype=torch.uint8, device=device)
    return buf.data_ptr(), buf


def _here() -> int:
    """The current device; -1 where there is none."""
    try:
        return torch.cuda.current_device() if kernels._raw_device is None else kernels._raw_device()
    except RuntimeError:
        return -1


def _seen(t: torch.Tensor) -> tuple:
    """What of a tensor a check may ask for."""
    return t.shape, t.stride(), t.dtype, t.get_device(), t.data_ptr() & 15


# ---- checks ----------------------------------------------------------------------------------------------------
def _on_device(what: str, *tensors) -> None:
    at = [t.get_device() for t in tensors if t is not None]
    if min(at) < 0:
        raise KernelError(f"{what}: a tensor that is not on a CUDA device (there is no CPU path)")
    here = _here()
    if min(at) != here or max(at) != here:
        raise KernelError(f"{what}: tensors on the devices {sorted(set(at))}, while the current device is {here}")


def _check_counts(what: str, *counts) -> None:
    """Rows, columns and pairs are 32-bit numbers in the launchers."""
    if max(counts) >= 2 ** 31:
        raise KernelError(f"{what}: {max(counts)} are too many for one call")


def _check_rows(what: str, rows: Fp8Rows, k: int, written: bool = False) -> None:
    q, s = rows
    kb = blocks_of(k)
    if q.dtype != F8 or q.dim() != 2 or q.shape[1] != kb * BLOCK or q.stride(1) != 1 or q.stride(0) % 16 or q.data_ptr() % 16 or \
            (q.shape[0] > 1 and q.stride(0) < kb * BLOCK):
        raise KernelError(f"{what}: quantised rows of {k} values are float8_e4m3fn [rows, {kb * BLOCK}], every row on 16 bytes; got "
                          f"{q.dtype} {list(q.shape)} with strides {list(q.stride())}")
    if s.dtype != torch.float32 or tuple(s.shape) != (kb, q.shape[0]) or (s.shape[1] > 1 and s.stride(1) != 1):
        raise KernelError(f"{what}: the rows' scales are float32 [{kb}, {q.shape[0]}], rows innermost; got {s.dtype} {list(s.shape)}")
    if written and kb > 1 and s.stride(0) < s.shape[1]:
        raise KernelError(f"{what}: the rows' scales that are written do not overlap; got {list(s.shape)} with strides {list(s.stride())}")


def _check_matrix(what: str, w: Fp8Matrix, gated: bool, stacked: bool) -> None:
    q, s, k = w
    kb, lead = blocks_of(k), q.shape[:1] if stacked else ()
    if k < 1:
        raise KernelError(f"{what}: a matrix of {k} columns")
    if q.dtype != F8 or q.dim() != 2 + stacked or q.shape[-1] != kb * BLOCK or not q.is_contiguous() or q.data_ptr() % 16:
        raise KernelError(f"{what}: a matrix of {k} columns in 8 bits is contiguous float8_e4m3fn [{'experts, ' if stacked else ''}rows, "
                          f"{kb * BLOCK}] on 16 bytes; got {q.dtype} {list(q.shape)}")
    n = q.shape[-2]
    if gated and n % 16:
        raise KernelError(f"{what}: gate and up rows come in eights; got {n} rows")
    shape = tuple(lead) + ((2, blocks_of(n // 2), kb) if gated else (blocks_of(n), kb))
    if s.dtype != torch.float32 or tuple(s.shape) != shape or not s.is_contiguous():
        raise KernelError(f"{what}: the matrix's scales are contiguous float32 {list(shape)}; got {s.dtype} {list(s.shape)}")


# ---- rows and matrices -----------------------------------------------------------------------------------------
def quantize_rows(x: torch.Tensor, rows: Fp8Rows, pair_row: Optional[torch.Tensor] = None) -> None:
    """``rows`` = x [T, K] (float32 or bfloat16) in 8 bits, a scale for every row and 128 columns; zeros behind K.
    ``pair_row`` int32 [T, top]: row t goes to the rows ``pair_row[t]`` instead (those below zero: nowhere)."""
    q, scale = rows
    key = (_seen(x), _seen(q), _seen(scale), None if pair_row is None else _seen(pair_row), _here())
    plan = _plans.get(key) or _plan_rows(key, x, rows, pair_row)
    f, given = plan
    rc = f(x.data_ptr(), *given[0], q.data_ptr(), given[1], scale.data_ptr(), given[2], None if pair_row is None else pair_row.data_ptr(), given[3], given[4],
           _stream())
    if rc:
        _failed(f)
    kernels.count_launches(1)


def _plan_rows(key, x, rows: Fp8Rows, pair_row) -> tuple:
    if x.dim() != 2 or (x.shape[1] > 1 and x.stride(1) != 1):
        raise KernelError("quantize_rows: rows of neighbouring values")
    tokens, k = x.shape
    if k < 1:
        raise KernelError("quantize_rows: rows without values")
    _check_counts("quantize_rows", tokens, k, rows.q.shape[0])
    _check_rows("quantize_rows", rows, k, written=True)
    top = 1
    if pair_row is not None:
        top = pair_row.numel() // max(tokens, 1)
        if pair_row.dtype != torch.int32 or not pair_row.is_contiguous() or pair_row.numel() != tokens * top:
            raise KernelError(f"quantize_rows: places are contiguous int32 [{tokens}, choices]")
    elif rows.q.shape[0] != tokens:
        raise KernelError(f"quantize_rows: {tokens} rows into {rows.q.shape[0]}")
    _on_device("quantize_rows", x, rows.q, rows.scale, pair_row)
    f = _f("g2b_quantize_rows", [c_void_p, c_int, c_longlong, c_int, c_int, c_void_p, c_longlong, c_void_p, c_longlong, c_void_p, c_int, c_int, c_void_p])
    if len(_plans) > 4096:
        _plans.clear()
    plan = _plans[key] = (f, ((_code(x.dtype), x.stride(0), tokens, k), rows.q.stride(0), rows.scale.stride(0), top, rows.q.shape[0]))
    return plan


def quantize_matrix(w: torch.Tensor) -> Fp8Matrix:
    """A matrix [N, K], or a stack [E, N, K], in 8 bits with a scale for every 128 x 128."""
    if w.dim() not in (2, 3) or not w.is_contiguous() or 0 in w.shape:
        raise KernelError("quantize_matrix: a contiguous matrix, or a stack of them, that is not empty")
    _check_counts("quantize_matrix", *w.shape)
    _on_device("quantize_matrix", w)
    n, k = w.shape[-2:]
    lead = tuple(w.shape[:-2])
    q = torch.empty(lead + (n, blocks_of(k) * BLOCK), dtype=F8, device=w.device)
    scale = torch.empty(lead + (blocks_of(n), blocks_of(k)), dtype=torch.float32, device=w.device)
    f = _f("g2b_quantize_matrix", [c_void_p, c_int, c_int, c_int, c_int, c_longlong, c_void_p, c_longlong, c_void_p, c_void_p])
    _call(f, _ptr(w), _code(w.dtype), lead[0] if lead else 1, n, k, k, _ptr(q), q.shape[-1], _ptr(scale), _stream())
    return Fp8Matrix(q, scale, k)


def stored_matrix(q: torch.Tensor, scale: torch.Tensor) -> Fp8Matrix:
    """A checkpoint's matrix and the scales of its blocks; rows are filled up with zeros to whole blocks."""
    if q.dim() != 2 or q.dtype != F8 or tuple(scale.shape) != (blocks_of(q.shape[0]), blocks_of(q.shape[1])) or not scale.is_floating_point():
        raise KernelError(f"stored_matrix: float8_e4m3fn [N, K] goes with a scale for every {BLOCK} x {BLOCK}; got {q.dtype} {list(q.shape)} and "
                          f"{scale.dtype} {list(scale.shape)}")
    k = q.shape[1]
    if k % BLOCK:
        q = torch.nn.functional.pad(q.view(torch.uint8), (0, blocks_of(k) * BLOCK - k)).view(F8)
    return Fp8Matrix(q.contiguous(), scale.to(torch.float32).contiguous(), k)


def gate_up_matrix(gate: Fp8Matrix, up: Fp8Matrix) -> Fp8Matrix:
    """Gate and up as one matrix, rows alternating in eights; the scales stay their own matrix's."""
    n = gate.q.shape[0]
    if gate.q.dim() != 2 or gate.scale.dim() != 2 or gate.k != up.k or up.q.shape != gate.q.shape or up.scale.shape != gate.scale.shape or n % 8:
        raise KernelError(f"gate_up_matrix: two matrices of one size, rows a multiple of 8; got {list(gate.shape)} and {list(up.shape)}")
    both = torch.stack([m.q.view(torch.uint8).reshape(n // 8, 8, -1) for m in (gate, up)], dim=1).reshape(2 * n, -1)
    return Fp8Matrix(both.view(F8), torch.stack([gate.scale, up.scale]).contiguous(), gate.k)


def no_matrix(n: int, k: int, device) -> Fp8Matrix:
    """Zeros."""
    return Fp8Matrix(torch.zeros((n, blocks_of(k) * BLOCK), dtype=torch.uint8, device=device).view(F8),
                     torch.ones((blocks_of(n), blocks_of(k)), dtype=torch.float32, device=device), k)


def stack_matrices(matrices) -> Fp8Matrix:
    """Matrices of one size as a stack (experts)."""
    matrices = list(matrices)
    if not matrices or any(m.q.dim() != 2 or m.k != matrices[0].k or m.q.shape != matrices[0].q.shape or m.scale.shape != matrices[0].scale.shape
                           for m in matrices):
        raise KernelError(f"stack_matrices: matrices of one size; got {[list(m.shape) for m in matrices[:4]]}")
    q = torch.stack([m.q.view(torch.uint8) for m in matrices])
    return Fp8Matrix(q.view(F8), torch.stack([m.scale for m in matrices]).contiguous(), matrices[0].k)


def side_by_side(matrices):
    """Matrices that read the same input as one, their outputs side by side; where one ends inside a block of 128 rows they stay apart."""
    if len(matrices) == 1:
        return matrices[0]
    if all(m.q.shape[0] % BLOCK == 0 for m in matrices[:-1]):
        return Fp8Matrix(torch.cat([m.q.view(torch.uint8) for m in matrices]).view(F8), torch.cat([m.scale for m in matrices]).contiguous(),
                         matrices[0].k)
    return Fp8Matrices(tuple(matrices))


# ---- products --------------------------------------------------------------------------------------------------
def _check_out(what: str, out: torch.Tensor, rows: int, columns: int) -> None:
    if tuple(out.shape) != (rows, columns) or (columns > 1 and out.stride(1) != 1) or (rows > 1 and out.stride(0) < columns):
        raise KernelError(f"{what}: the output is [{rows}, {columns}], rows of neighbouring values that do not overlap; got {list(out.shape)} with "
                          f"strides {list(out.stride())}")


def _check_values(what: str, a: torch.Tensor, k: int) -> None:
    if a.dim() != 2 or a.shape[1] != k or a.dtype not in (torch.float32, torch.bfloat16) or (k > 1 and a.stride(1) != 1):
        raise KernelError(f"{what}: {a.dtype} {list(a.shape)} with strides {list(a.stride())} against a matrix of {k} columns; rows of neighbouring "
                          "float32 or bfloat16 values")


def _plan_product(key, what: str, a, w: Fp8Matrix, out, epi: int, form, columns: int, split: int, defines) -> _Plan:
    """Checks everything that a product's kernels rely on; ``epi`` below zero: whichever store the output's type asks for."""
    gated = epi in (EPI_GATED_F32, EPI_GATED_ROWS)
    as_rows, given = isinstance(out, Fp8Rows), isinstance(a, Fp8Rows)
    _check_matrix(what, w, gated, False)
    tokens = (a.q if given else a).shape[0]
    _check_counts(what, tokens, w.q.shape[0], w.k)
    n = w.q.shape[0] // 2 if gated else w.q.shape[0]
    if as_rows:
        _check_rows(what, out, n, written=True)
        if out.q.shape[0] != tokens:
            raise KernelError(f"{what}: {tokens} rows into {out.q.shape[0]}")
    else:
        _check_out(what, out, tokens, n)
    if given:
        _check_rows(what, a, w.k)
    else:
        _check_values(what, a, w.k)
    _on_device(what, *(a if given else (a,)), w.q, w.scale, *(out if as_rows else (out,)))
    call, to = _Call(), out.q if as_rows else out
    call.M, call.N, call.K, call.epi = tokens, w.q.shape[0], w.k, epi
    call.columns, call.split, call.with_x = 16 if columns == WITH_X else columns, split, 1 if columns == WITH_X else 0
    call.ldw, call.ldo, call.ldos = w.q.shape[1], to.stride(0), out.scale.stride(0) if as_rows else 0
    call.limit, call.offset, call.c1, call.c3 = form
    if given:
        call.x_dtype, call.lda, call.lds = -1, a.q.stride(0), a.scale.stride(0)
    else:
        call.x_dtype, call.x_stride = _code(a.dtype), a.stride(0)
    return _plan(key, call, w.q.device, "g2b_fp8_product_plan", "g2b_fp8_product", [c_void_p] * 10, not given and a.data_ptr() % 16 == 0,
                 columns == BY_THE_RULE, defines)


def _product(what: str, a, w: Fp8Matrix, out, epi: int, form=SILU, workspace=None, columns: int = BY_THE_RULE, split: int = 1, defines=()) -> None:
    """``columns`` and ``split``: the tiles of ``gemm_fp8_few.cuh`` and the parts of K (``BY_THE_RULE``: what ``choose`` in products_fp8.cu says)."""
    q, s, k = w
    if a.__class__ is Fp8Rows:
        x, x_scale = a
        seen = _seen(x_scale)
    else:
        x, x_scale, seen = a, None, None
    if out.__class__ is Fp8Rows:
        to, to_scale = out
        seen = (seen, _seen(to_scale))
    else:
        to, to_scale = out, None
    at_x, at_q, at_to = x.data_ptr(), q.data_ptr(), to.data_ptr()
    key = (x.shape, x.stride(), x.dtype, x.get_device(), at_x & 15, q.shape, q.stride(), q.dtype, q.get_device(), at_q & 15, s.shape, s.stride(), s.dtype,
           s.get_device(), to.shape, to.stride(), to.dtype, to.get_device(), at_to & 15, k, seen, epi, form, _here(), columns, split, defines)
    plan = _plans.get(key)
    if plan is None:
        plan = _plan_product(key, what, a, w, out, epi, form, columns, split, defines)
    scratch = held = None
    if plan.scratch or workspace is not None:
        scratch, held = _scratch(plan, workspace, "fp8.product", q.device)
    n = plan.f(plan.at, at_x, None if x_scale is None else x_scale.data_ptr(), scratch, at_q, s.data_ptr(), at_to,
               None if to_scale is None else to_scale.data_ptr(), plan.status, _stream())
    if n < 0:
        _failed(plan.f)
    kernels.count_launches(n)


def linear(a, w, out: torch.Tensor, accumulate: bool, workspace) -> None:
    if w.__class__ is Fp8Matrices:
        rows, at = a, 0
        _check_out("linear", out, (a.q if isinstance(a, Fp8Rows) else a).shape[0], w.shape[0])
        if not isinstance(a, Fp8Rows):                   # quantised once for all of them
            _check_values("linear", a, w.parts[0].k)
            rows = new_rows(a.shape[0], w.parts[0].k, workspace, "fp8.rows", a.device)
            quantize_rows(a, rows)
        for part in w.parts:
            n = part.q.shape[0]
            linear(rows, part, out[:, at:at + n], accumulate, workspace)
            at += n
        return
    if out.dtype == torch.float32:
        epi = EPI_ADD_F32 if accumulate else EPI_F32
    elif out.dtype == torch.bfloat16 and not accumulate:
        epi = EPI_BF16
    else:
        raise KernelError(f"linear: stores float32 or bfloat16 and adds to float32; got {out.dtype}")
    _product("linear", a, w, out, epi, SILU, workspace)


def gate_up(a, w: Fp8Matrix, mid, form, workspace) -> None:
    """mid = glu(gate, up) of a @ w.T, in float32 [T, I], or quantised (``Fp8Rows``)."""
    if isinstance(mid, Fp8Rows):
        return _product("gate_up_fused", a, w, mid, EPI_GATED_ROWS, form, workspace)
    if mid.dtype != torch.float32:
        raise KernelError(f"gate_up_fused: a matrix in 8 bits leaves float32 or quantised rows, not {mid.dtype}")
    _product("gate_up_fused", a, w, mid, EPI_GATED_F32, form, workspace)


# ---- experts ---------------------------------------------------------------------------------------------------
def moe_sort(idx: torch.Tensor, n_real: int, starts: torch.Tensor, pair_row: torch.Tensor, row_pair: Optional[torch.Tensor] = None) -> None:
    """Rows for the (token, choice) pairs of ``idx``, expert by expert and within an expert in their order: ``starts`` int32 [n_real + 1],
    ``pair_row`` int32 like idx (-1: an expert from ``n_real`` on); ``row_pair``, where given: the pair of every row that one has."""
    for t, what, n in ((idx, "idx", idx.numel()), (starts, "starts", n_real + 1), (pair_row, "pair_row", idx.numel()), (row_pair, "row_pair", idx.numel())):
        if t is None:
            continue
        if t.dtype != torch.int32 or not t.is_contiguous() or t.numel() != n:
            raise KernelError(f"moe_sort: {what} is contiguous int32 of {n}; got {t.dtype} {list(t.shape)}")
    _check_counts("moe_sort", idx.numel() + SORTED_AT_ONCE, n_real)
    _on_device("moe_sort", idx, starts, pair_row, row_pair)
    f = _f("g2b_moe_sort", [c_void_p, c_int, c_int, c_void_p, c_void_p, c_void_p, c_void_p])
    _call(f, _ptr(idx), idx.numel(), n_real, _ptr(starts), _ptr(pair_row), _ptr(row_pair), _stream())


def _plan_experts(key, h, idx, w_gate_up: Fp8Matrix, w_down: Fp8Matrix, rows32, pair_row, form, forced) -> _Plan:
    what = "moe_experts_fp8"
    _check_matrix(what, w_gate_up, True, True)
    _check_matrix(what, w_down, False, True)
    n_experts, inter = w_gate_up.q.shape[0], w_gate_up.q.shape[1] // 2
    if w_down.k != inter or w_down.q.shape[0] != n_experts:
        raise KernelError(f"{what}: gate and up of {n_experts} experts with {inter} outputs against down matrices {list(w_down.q.shape)} of "
                          f"{w_down.k} columns")
    _check_values(what, h, w_gate_up.k)
    if idx.dim() != 2 or idx.shape[0] != h.shape[0] or idx.dtype != torch.int32 or not idx.is_contiguous():
        raise KernelError(f"{what}: choices are contiguous int32 [{h.shape[0]}, top]; got {idx.dtype} {list(idx.shape)}")
    if n_experts > MOST_EXPERTS:
        raise KernelError(f"{what}: {n_experts} experts, at most {MOST_EXPERTS}")
    n_pairs = idx.numel()
    _check_counts(what, h.shape[0], n_pairs + SORTED_AT_ONCE, w_gate_up.q.shape[1], w_gate_up.k, w_down.q.shape[1])
    if rows32.dtype != torch.float32 or tuple(rows32.shape) != (n_pairs, w_down.q.shape[1]) or not rows32.is_contiguous():
        raise KernelError(f"{what}: the experts' rows are contiguous float32 [{n_pairs}, {w_down.q.shape[1]}]")
    if pair_row.dtype != torch.int32 or pair_row.numel() != n_pairs or not pair_row.is_contiguous():
        raise KernelError(f"{what}: pair_row is contiguous int32 of {n_pairs}")
    _on_device(what, h, idx, w_gate_up.q, w_gate_up.scale, w_down.q, w_down.scale, rows32, pair_row)
    call = _Call()
    call.M, call.N, call.K, call.x_dtype, call.n_experts = h.shape[0], 2 * inter, w_gate_up.k, _code(h.dtype), n_experts
    call.top, call.H, call.x_stride, call.ldw = idx.shape[1], w_down.q.shape[1], h.stride(0), w_gate_up.q.shape[2]
    call.limit, call.offset, call.c1, call.c3 = form
    if forced is not None:
        (columns, call.split), (columns_2, call.split_2) = forced
        call.columns, call.with_x = (16, 1) if columns == WITH_X else (columns, 0)
        call.columns_2, call.with_x_2 = (16, 1) if columns_2 == WITH_X else (columns_2, 0)
        if call.with_x != call.with_x_2:
            raise KernelError(f"{what}: both products quantise their rows, or neither does")
    return _plan(key, call, h.device, "g2b_fp8_experts_plan", "g2b_fp8_experts", [c_void_p] * 12, h.data_ptr() % 16 == 0, forced is None)


def moe_experts(h: torch.Tensor, idx: torch.Tensor, w_gate_up: Fp8Matrix, w_down: Fp8Matrix, rows32: torch.Tensor, pair_row: torch.Tensor, form,
                workspace, forced=None) -> None:
    """``forced``: the (columns, parts) of the gated and of the down products, as ``_product`` has them (None: what ``choose`` says)."""
    gq, gs, gk = w_gate_up
    dq, ds, dk = w_down
    key = (_seen(h), _seen(idx), _seen(gq), _seen(gs), gk, _seen(dq), _seen(ds), dk, _seen(rows32), _seen(pair_row), form, _here(), forced)
    plan = _plans.get(key) or _plan_experts(key, h, idx, w_gate_up, w_down, rows32, pair_row, form, forced)
    scratch, held = _scratch(plan, workspace, "fp8.experts", gq.device)
    n = plan.f(plan.at, h.data_ptr(), idx.data_ptr(), scratch, gq.data_ptr(), gs.data_ptr(), dq.data_ptr(), ds.data_ptr(), rows32.data_ptr(),
               pair_row.data_ptr(), plan.status, _stream())
    if n < 0:
        _failed(plan.f)
    kernels.count_launches(n)


def moe_back(rows32, pair_row, weight, x_self, out, accumulate: bool) -> None:
    key = (_seen(rows32), _seen(pair_row), _seen(weight), _seen(x_self), _seen(out), accumulate, _here())
    f, given = _plans.get(key) or _plan_back(key, rows32, pair_row, weight, x_self, out, accumulate)
    rc = f(rows32.data_ptr(), pair_row.data_ptr(), weight.data_ptr(), x_self.data_ptr(), *given[0], out.data_ptr(), *given[1], _stream())
    if rc:
        _failed(f)
    kernels.count_launches(1)


def _plan_back(key, rows32, pair_row, weight, x_self, out, accumulate: bool) -> tuple:
    if weight.dim() != 2 or out.dim() != 2:
        raise KernelError("moe_back: weights [tokens, top] and an output [tokens, width]")
    tokens, top = weight.shape
    width = out.shape[1]
    _check_counts("moe_back", tokens, top, width, rows32.shape[0])
    if weight.dtype != torch.float32 or not weight.is_contiguous() or pair_row.dtype != torch.int32 or not pair_row.is_contiguous() or \
            pair_row.numel() != tokens * top:
        raise KernelError(f"moe_back: weights are contiguous float32 [{tokens}, {top}], rows of the pairs as many int32")
    if rows32.dtype != torch.float32 or not rows32.is_contiguous() or rows32.dim() != 2 or rows32.shape[1] != width:
        raise KernelError(f"moe_back: the experts' rows are contiguous float32 [pairs, {width}]")
    _check_out("moe_back", out, tokens, width)
    _check_out("moe_back", x_self, tokens, width)
    if accumulate and out.dtype != torch.float32:
        raise KernelError("moe_back: only a float32 output is added to")
    _on_device("moe_back", rows32, pair_row, weight, x_self, out)
    f = _f("g2b_moe_back", [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_longlong, c_int, c_int, c_int, c_int, c_void_p, c_int, c_longlong, c_int, c_void_p])
    if len(_plans) > 4096:
        _plans.clear()
    plan = _plans[key] = (f, ((_code(x_self.dtype), x_self.stride(0), rows32.shape[0], tokens, top, width), (_code(out.dtype), out.stride(0), 1 if accumulate else 0)))
    return plan
