"""Bindings of the kernels in 8-bit floating point (``csrc/fp8.cuh`` says how values are held)."""
from __future__ import annotations

from ctypes import c_float, c_int, c_longlong, c_void_p
from typing import Optional

import torch

from . import kernels
from .kernels_bf16 import _status_word
from .kernels import SILU, Fp8Matrices, Fp8Matrix, Fp8Rows, KernelError, _call, _code, _fn, _ptr, _stream

BLOCK = 128                          # values of a row, and of either side of a matrix, that share a scale
F8 = torch.float8_e4m3fn
MOST_EXPERTS = 1024                  # csrc/quant_fp8.cu
EPI_BF16, EPI_F32, EPI_ADD_F32, EPI_GATED_F32, EPI_GATED_ROWS = 0, 1, 2, 3, 4
_FORM = [c_float] * 4


def blocks_of(n: int) -> int:
    return -(-n // BLOCK)


def new_rows(tokens: int, k: int, workspace, name: str, device) -> Fp8Rows:
    """Room for the quantised rows of ``tokens`` times ``k`` values: of the workspace, or, without one, new."""
    kb = blocks_of(k)
    if workspace is None:
        return Fp8Rows(torch.empty((tokens, kb * BLOCK), dtype=F8, device=device),
                       torch.empty((kb, tokens), dtype=torch.float32, device=device))
    return Fp8Rows(workspace.buffer(name + ".q", (tokens, kb * BLOCK), F8), workspace.buffer(name + ".scale", (kb, tokens), torch.float32))


# ---- checks ----------------------------------------------------------------------------------------------------
def _on_device(what: str, *tensors) -> None:
    at = [t.get_device() for t in tensors if t is not None]
    if min(at) < 0:
        raise KernelError(f"{what}: a tensor that is not on a CUDA device (there is no CPU path)")
    here = torch.cuda.current_device() if kernels._raw_device is None else kernels._raw_device()
    if min(at) != here or max(at) != here:
        raise KernelError(f"{what}: tensors on the devices {sorted(set(at))}, while the current device is {here}")


def _check_rows(what: str, rows: Fp8Rows, k: int) -> None:
    q, s = rows
    kb = blocks_of(k)
    if q.dtype != F8 or q.dim() != 2 or q.shape[1] != kb * BLOCK or q.stride(1) != 1 or q.stride(0) % 16 or q.data_ptr() % 16 or \
            (q.shape[0] > 1 and q.stride(0) < kb * BLOCK):
        raise KernelError(f"{what}: quantised rows of {k} values are float8_e4m3fn [rows, {kb * BLOCK}], every row on 16 bytes; got "
                          f"{q.dtype} {list(q.shape)} with strides {list(q.stride())}")
    if s.dtype != torch.float32 or tuple(s.shape) != (kb, q.shape[0]) or (s.shape[1] > 1 and s.stride(1) != 1):
        raise KernelError(f"{what}: the rows' scales are float32 [{kb}, {q.shape[0]}], rows innermost; got {s.dtype} {list(s.shape)}")


def _check_matrix(what: str, w: Fp8Matrix, gated: bool, stacked: bool) -> None:
    q, s, k = w
    kb, lead = blocks_of(k), q.shape[:1] if stacked else ()
    if q.dtype != F8 or q.dim() != 2 + stacked or q.shape[-1] != kb * BLOCK or not q.is_contiguous() or q.data_ptr() % 16:
        raise KernelError(f"{what}: a matrix of {k} columns in 8 bits is contiguous float8_e4m3fn [{'experts, ' if stacked else ''}rows, "
                          f"{kb * BLOCK}] on 16 bytes; got {q.dtype} {list(q.shape)}")
    n = q.shape[-2]
    if gated and n % 16:
        raise KernelError(f"{what}: gate and up rows come in eights; got {n} rows")
    shape = tuple(lead) + ((2, blocks_of(n // 2), kb) if gated else (blocks_of(n), kb))
    if s.dtype != torch.float32 or tuple(s.shape) != shape or not s.is_contiguous():
        raise KernelError(f"{what}: the matrix's scales are contiguous float32 {list(shape)}; got {s.dtype} {list(s.shape)}")


def _quantised(what: str, a, k: int, workspace, name: str = "fp8.rows") -> Fp8Rows:
    if isinstance(a, Fp8Rows):
        _check_rows(what, a, k)
        return a
    if a.dim() != 2 or a.shape[1] != k:
        raise KernelError(f"{what}: {list(a.shape)} values against a matrix of {k} columns")
    rows = new_rows(a.shape[0], k, workspace, name, a.device)
    quantize_rows(a, rows)
    return rows


# ---- rows and matrices -----------------------------------------------------------------------------------------
def quantize_rows(x: torch.Tensor, rows: Fp8Rows, pair_row: Optional[torch.Tensor] = None) -> None:
    """``rows`` = x [T, K] (float32 or bfloat16) in 8 bits, a scale for every row and 128 columns; zeros behind K.
    ``pair_row`` int32 [T, top]: row t goes to the rows ``pair_row[t]`` instead (those below zero: nowhere)."""
    if x.dim() != 2 or (x.shape[1] > 1 and x.stride(1) != 1):
        raise KernelError("quantize_rows: rows of neighbouring values")
    tokens, k = x.shape
    if k < 1:
        raise KernelError("quantize_rows: rows without values")
    _check_rows("quantize_rows", rows, k)
    top = 1
    if pair_row is not None:
        top = pair_row.numel() // max(tokens, 1)
        if pair_row.dtype != torch.int32 or not pair_row.is_contiguous() or pair_row.numel() != tokens * top:
            raise KernelError(f"quantize_rows: places are contiguous int32 [{tokens}, choices]")
    elif rows.q.shape[0] != tokens:
        raise KernelError(f"quantize_rows: {tokens} rows into {rows.q.shape[0]}")
    _on_device("quantize_rows", x, rows.q, rows.scale, pair_row)
    if tokens == 0:
        return
    f = _fn("quant_fp8.cu", "g2b_quantize_rows", [c_void_p, c_int, c_longlong, c_int, c_int, c_void_p, c_longlong, c_void_p, c_longlong, c_void_p,
                                                  c_int, c_int, c_void_p])
    _call(f, _ptr(x), _code(x.dtype), x.stride(0), tokens, k, _ptr(rows.q), rows.q.stride(0), _ptr(rows.scale), rows.scale.stride(0),
          _ptr(pair_row), top, rows.q.shape[0], _stream())


def quantize_matrix(w: torch.Tensor) -> Fp8Matrix:
    """A matrix [N, K], or a stack [E, N, K], in 8 bits with a scale for every 128 x 128."""
    if w.dim() not in (2, 3) or not w.is_contiguous() or 0 in w.shape:
        raise KernelError("quantize_matrix: a contiguous matrix, or a stack of them, that is not empty")
    _on_device("quantize_matrix", w)
    n, k = w.shape[-2:]
    lead = tuple(w.shape[:-2])
    q = torch.empty(lead + (n, blocks_of(k) * BLOCK), dtype=F8, device=w.device)
    scale = torch.empty(lead + (blocks_of(n), blocks_of(k)), dtype=torch.float32, device=w.device)
    f = _fn("quant_fp8.cu", "g2b_quantize_matrix", [c_void_p, c_int, c_int, c_int, c_int, c_longlong, c_void_p, c_longlong, c_void_p, c_void_p])
    _call(f, _ptr(w), _code(w.dtype), lead[0] if lead else 1, n, k, k, _ptr(q), q.shape[-1], _ptr(scale), _stream())
    return Fp8Matrix(q, scale, k)


def stored_matrix(q: torch.Tensor, scale: torch.Tensor) -> Fp8Matrix:
    """A checkpoint's matrix and the scales of its blocks; rows are filled up with zeros to whole blocks."""
    n, k = q.shape
    if q.dtype != F8 or tuple(scale.shape) != (blocks_of(n), blocks_of(k)):
        raise KernelError(f"stored_matrix: float8_e4m3fn [{n}, {k}] goes with scales [{blocks_of(n)}, {blocks_of(k)}]; got {q.dtype} and "
                          f"{list(scale.shape)}")
    if k % BLOCK:
        q = torch.nn.functional.pad(q.view(torch.uint8), (0, blocks_of(k) * BLOCK - k)).view(F8)
    return Fp8Matrix(q.contiguous(), scale.to(torch.float32).contiguous(), k)


def gate_up_matrix(gate: Fp8Matrix, up: Fp8Matrix) -> Fp8Matrix:
    """Gate and up as one matrix, rows alternating in eights; the scales stay their own matrix's."""
    n = gate.q.shape[0]
    if gate.k != up.k or up.q.shape[0] != n or n % 8:
        raise KernelError(f"gate_up_matrix: two matrices of one size, rows a multiple of 8; got {list(gate.q.shape)} and {list(up.q.shape)}")
    both = torch.stack([m.q.view(torch.uint8).view(n // 8, 8, -1) for m in (gate, up)], dim=1).reshape(2 * n, -1)
    return Fp8Matrix(both.view(F8), torch.stack([gate.scale, up.scale]).contiguous(), gate.k)


def stack_matrices(matrices) -> Fp8Matrix:
    """Matrices of one size as a stack (experts)."""
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
def _product_tc(rows: Fp8Rows, w: Fp8Matrix, out, epi: int, form, starts, workspace, defines=()) -> None:
    """``out``: a tensor, or ``Fp8Rows`` with ``EPI_GATED_ROWS``."""
    as_rows = epi == EPI_GATED_ROWS
    to, scale = out if as_rows else (out, None)
    if workspace is not None:
        workspace.waits = True
    f = _fn("gemm_fp8_tc.cu", "g2b_gemm_fp8_tc",
            [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_longlong, c_longlong, c_longlong, c_longlong,
             c_longlong, c_int, *_FORM, c_void_p, c_int, c_void_p, c_void_p], defines=tuple(defines))
    _call(f, _ptr(rows.q), _ptr(rows.scale), _ptr(w.q), _ptr(w.scale), _ptr(to), _ptr(scale), rows.q.shape[0], w.q.shape[-2], blocks_of(w.k),
          rows.q.stride(0), rows.scale.stride(0), w.q.shape[-1], to.stride(0), scale.stride(0) if as_rows else 0, epi, *form, _ptr(starts),
          w.q.shape[0] if starts is not None else 0, _ptr(_status_word(to.device)), _stream())


def _product_few(rows: Fp8Rows, w: Fp8Matrix, out, epi: int, form, starts, workspace, columns: int, split: int, defines=()) -> None:
    """``columns`` (16, 32, 64 or 128) rows of activations side by side in a tile (-128: 128 on the lanes of tensor memory, beside 128 rows of the matrix),
    K in ``split`` parts, at most 8."""
    if workspace is not None:
        workspace.waits = True
    f = _fn("gemm_fp8_few.cu", "g2b_gemm_fp8_few",
            [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_longlong, c_longlong, c_longlong, c_longlong, c_int, *_FORM,
             c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_void_p], defines=tuple(defines))
    _call(f, _ptr(rows.q), _ptr(rows.scale), _ptr(w.q), _ptr(w.scale), _ptr(out), rows.q.shape[0], w.q.shape[-2], blocks_of(w.k),
          rows.q.stride(0), rows.scale.stride(0), w.q.shape[-1], out.stride(0), epi, *form, _ptr(starts), w.q.shape[0] if starts is not None else 0,
          abs(columns), 1 if columns < 0 else 0, split, _ptr(_status_word(out.device)), _stream())


MANY_ROWS = 128                      # rows (of an expert, on average) up to which a product goes to the kernel of few rows


def few_shape(rows: int, n: int, blocks: int, experts: int = 0) -> tuple:
    """(columns, parts of K) of the kernel of few rows."""
    each = -(-rows // experts) if experts else rows
    columns = next((c for c in (16, 32, 64) if each <= c), 128)
    tiles = -(-n // 128) * (min(experts, rows) if experts else -(-rows // columns))
    most = 296 if columns <= 32 else 148           # CTAs that are there at once
    split = 1
    while split < 8 and tiles * split * 2 <= most and blocks >= 4 * split:
        split *= 2
    return columns, split


def _product(rows: Fp8Rows, w: Fp8Matrix, out: torch.Tensor, epi: int, form=SILU, starts=None, workspace=None) -> None:
    stacked, n = starts is not None, rows.q.shape[0]
    if n > MANY_ROWS * (w.q.shape[0] if stacked else 1):
        return _product_tc(rows, w, out, epi, form, starts, workspace)
    if epi == EPI_GATED_ROWS:
        inter = w.q.shape[-2] // 2
        h = torch.empty((n, inter), dtype=torch.float32, device=w.q.device) if workspace is None else \
            workspace.buffer("fp8.mid", (n, inter), torch.float32)
        _product(rows, w, h, EPI_GATED_F32, form, starts, workspace)
        return quantize_rows(h, out)
    _product_few(rows, w, out, epi, form, starts, workspace, *few_shape(n, w.q.shape[-2], blocks_of(w.k), w.q.shape[0] if stacked else 0))


def _check_out(what: str, out: torch.Tensor, rows: int, columns: int) -> None:
    if tuple(out.shape) != (rows, columns) or (columns > 1 and out.stride(1) != 1) or (rows > 1 and out.stride(0) < columns):
        raise KernelError(f"{what}: the output is [{rows}, {columns}], rows of neighbouring values that do not overlap; got {list(out.shape)} with "
                          f"strides {list(out.stride())}")


def linear(a, w, out: torch.Tensor, accumulate: bool, workspace) -> None:
    if isinstance(w, Fp8Matrices):
        rows, at = _quantised("linear", a, w.parts[0].k, workspace), 0
        _check_out("linear", out, rows.q.shape[0], w.shape[0])
        for part in w.parts:
            n = part.q.shape[0]
            linear(rows, part, out[:, at:at + n], accumulate, workspace)
            at += n
        return
    _check_matrix("linear", w, False, False)
    tokens = a.q.shape[0] if isinstance(a, Fp8Rows) else a.shape[0]
    _check_out("linear", out, tokens, w.q.shape[0])
    if out.dtype not in (torch.float32, torch.bfloat16) or (accumulate and out.dtype != torch.float32):
        raise KernelError(f"linear: stores float32 or bfloat16 and adds to float32; got {out.dtype}")
    rows = _quantised("linear", a, w.k, workspace)
    _on_device("linear", rows.q, rows.scale, w.q, w.scale, out)
    if tokens:
        _product(rows, w, out, EPI_ADD_F32 if accumulate else EPI_F32 if out.dtype == torch.float32 else EPI_BF16, workspace=workspace)


def gate_up(a, w: Fp8Matrix, mid, form, workspace) -> None:
    """mid = glu(gate, up) of a @ w.T, in float32 [T, I], or quantised (``Fp8Rows``)."""
    _check_matrix("gate_up_fused", w, True, False)
    tokens, inter = a.q.shape[0] if isinstance(a, Fp8Rows) else a.shape[0], w.q.shape[0] // 2
    as_rows = isinstance(mid, Fp8Rows)
    if as_rows:
        _check_rows("gate_up_fused", mid, inter)
        if mid.q.shape[0] != tokens:
            raise KernelError(f"gate_up_fused: {tokens} rows into {mid.q.shape[0]}")
    else:
        _check_out("gate_up_fused", mid, tokens, inter)
        if mid.dtype != torch.float32:
            raise KernelError(f"gate_up_fused: a matrix in 8 bits leaves float32 or quantised rows, not {mid.dtype}")
    rows = _quantised("gate_up_fused", a, w.k, workspace)
    _on_device("gate_up_fused", rows.q, rows.scale, w.q, w.scale, mid.q if as_rows else mid)
    if tokens:
        _product(rows, w, mid, EPI_GATED_ROWS if as_rows else EPI_GATED_F32, form, workspace=workspace)


# ---- experts ---------------------------------------------------------------------------------------------------
def moe_sort(idx: torch.Tensor, n_real: int, starts: torch.Tensor, pair_row: torch.Tensor) -> None:
    """Rows for the (token, choice) pairs of ``idx``, expert by expert and within an expert in their order: ``starts`` int32 [n_real + 1],
    ``pair_row`` int32 like idx (-1: an expert from ``n_real`` on)."""
    for t, what, n in ((idx, "idx", idx.numel()), (starts, "starts", n_real + 1), (pair_row, "pair_row", idx.numel())):
        if t.dtype != torch.int32 or not t.is_contiguous() or t.numel() != n:
            raise KernelError(f"moe_sort: {what} is contiguous int32 of {n}; got {t.dtype} {list(t.shape)}")
    _on_device("moe_sort", idx, starts, pair_row)
    f = _fn("quant_fp8.cu", "g2b_moe_sort", [c_void_p, c_int, c_int, c_void_p, c_void_p, c_void_p])
    _call(f, _ptr(idx), idx.numel(), n_real, _ptr(starts), _ptr(pair_row), _stream())


def moe_experts(h: torch.Tensor, idx: torch.Tensor, w_gate_up: Fp8Matrix, w_down: Fp8Matrix, rows32: torch.Tensor, pair_row: torch.Tensor, form,
                workspace) -> None:
    what = "moe_experts_fp8"
    _check_matrix(what, w_gate_up, True, True)
    _check_matrix(what, w_down, False, True)
    n_experts, inter = w_gate_up.q.shape[0], w_gate_up.q.shape[1] // 2
    if w_down.k != inter or w_down.q.shape[0] != n_experts:
        raise KernelError(f"{what}: gate and up of {n_experts} experts with {inter} outputs against down matrices {list(w_down.q.shape)} of "
                          f"{w_down.k} columns")
    if h.dim() != 2 or idx.dim() != 2 or idx.shape[0] != h.shape[0] or h.shape[1] != w_gate_up.k:
        raise KernelError(f"{what}: tokens {list(h.shape)} and choices {list(idx.shape)} for matrices of {w_gate_up.k} columns")
    if n_experts > MOST_EXPERTS:
        raise KernelError(f"{what}: {n_experts} experts, at most {MOST_EXPERTS}")
    n_pairs = idx.numel()
    if rows32.dtype != torch.float32 or tuple(rows32.shape) != (n_pairs, w_down.q.shape[1]) or not rows32.is_contiguous():
        raise KernelError(f"{what}: the experts' rows are contiguous float32 [{n_pairs}, {w_down.q.shape[1]}]")
    _on_device(what, h, idx, w_gate_up.q, w_gate_up.scale, w_down.q, w_down.scale, rows32, pair_row)
    if not n_pairs:
        return

    def scratch(name, shape, dtype):
        return torch.empty(shape, dtype=dtype, device=h.device) if workspace is None else workspace.buffer(name, shape, dtype)

    starts = scratch("fp8.starts", (n_experts + 1,), torch.int32)
    moe_sort(idx, n_experts, starts, pair_row)
    rows = new_rows(n_pairs, w_gate_up.k, workspace, "fp8.sorted", h.device)
    quantize_rows(h, rows, pair_row)
    mid = new_rows(n_pairs, inter, workspace, "fp8.mid_rows", h.device)
    _product(rows, w_gate_up, mid, EPI_GATED_ROWS, form, starts, workspace)
    _product(mid, w_down, rows32, EPI_F32, SILU, starts, workspace)


def moe_back(rows32, pair_row, weight, x_self, out, accumulate: bool) -> None:
    tokens, top = weight.shape
    width = out.shape[-1]
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
    f = _fn("quant_fp8.cu", "g2b_moe_back", [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_longlong, c_int, c_int, c_int, c_int, c_void_p,
                                             c_int, c_longlong, c_int, c_void_p])
    _call(f, _ptr(rows32), _ptr(pair_row), _ptr(weight), _ptr(x_self), _code(x_self.dtype), x_self.stride(0), rows32.shape[0], tokens, top, width, _ptr(out),
          _code(out.dtype), out.stride(0), 1 if accumulate else 0, _stream())
