"""Layers in 8-bit integers: the residual's addition and RMSNorm with rows in 8 bits, rows to 8 bits, and the product of 8-bit rows with
8-bit channels. Torch tensors in, the C ABI underneath, in the manner of ``attention``.

The three are the linear part of a layer: ``rmsnorm_i8`` in front of the Q/K/V and the gate/up projection, ``quantize_i8`` in front of
the output and the down projection (and, at load time, over a weight matrix, whose rows are its channels), ``gemm_i8`` for
each projection, for one token or for all tokens of many prompts. ``model.Llama(weight_type="i8")`` runs them together.

An 8-bit matrix is an int8 tensor [rows, k] whose rows are a multiple of 16 bytes apart (``rows_i8`` makes one) beside fp32 scales [rows]:
row r stands for scale[r] * q[r].
"""
from __future__ import annotations

import struct

import torch

from . import binding as _b
from .attention import _DTYPES
from .context import _enqueue, _on, _one_device

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
MAX_K = 131071  # longest inner dimension of gemm_i8: 32-bit sums of products of 8 bits stay exact

# The argument structures as the library lays them out (packed: see context).
ROWS_ARGS = struct.Struct("@6P4Q2If2i0P")
GEMM_ARGS = struct.Struct("@5P3Q3I2iP")


def rows_i8(rows: int, k: int, device=None) -> torch.Tensor:
    """An int8 tensor [rows, k] laid out as the operators take it: rows k rounded up to a multiple of 16 bytes apart."""
    return torch.empty((rows, (k + 15) // 16 * 16), dtype=torch.int8, device="cuda" if device is None else device)[:, :k]


def _matrix(t: torch.Tensor, rows: int, dim: int, what: str) -> int:
    """Distance of the rows of a [rows, dim] tensor; 0, which the library takes as dense, where there is one."""
    if t.dim() != 2 or t.shape[0] != rows or t.shape[1] != dim:
        raise ValueError(f"{what} must be [{rows}, {dim}]")
    stride = t.stride()
    if dim > 1 and stride[1] != 1:
        raise ValueError(f"the rows of {what} must be dense")
    if rows < 2:
        return 0
    if stride[0] < dim:
        raise ValueError(f"the rows of {what} must not share memory (expanded or overlapping rows)")
    return stride[0]


def _bytes(q: torch.Tensor, rows: int, k: int, what: str) -> int:
    """Distance of the rows of an 8-bit matrix in bytes."""
    if q.dtype != torch.int8:
        raise TypeError(f"{what} must be int8")
    stride = _matrix(q, rows, k, what)
    if stride % 16:
        raise ValueError(f"the rows of {what} must be a multiple of 16 bytes apart (rows_i8 lays them out so)")
    return stride or (k + 15) // 16 * 16


def _scales(s: torch.Tensor, rows: int, what: str) -> int:
    if s.dtype != torch.float32 or s.dim() != 1 or s.shape[0] != rows or (rows > 1 and s.stride(0) != 1):
        raise ValueError(f"{what} must be a dense fp32 tensor [{rows}]")
    return s.data_ptr()


def _rows(entry: str, x, weight, eps: float, delta, x_out, out, scale, stream):
    index = _one_device(x, weight, delta, x_out, out, scale)
    if x.dim() != 2:
        raise ValueError("x must be [N, D]")
    N, D = x.shape
    x_dtype = x.dtype
    if x_dtype not in _FLOATS:
        raise TypeError("x must be fp32, fp16 or bf16")
    x_stride = _matrix(x, N, D, "x")
    weight_ptr = delta_ptr = delta_stride = delta_code = x_out_ptr = x_out_stride = 0
    if weight is not None:
        if weight.dtype != torch.float32 or weight.dim() != 1 or weight.shape[0] != D or not weight.is_contiguous():
            raise ValueError(f"weight must be a dense fp32 tensor [{D}]")
        weight_ptr = weight.data_ptr()
    if delta is not None:
        if delta.dtype not in _FLOATS:
            raise TypeError("delta must be fp32, fp16 or bf16")
        delta_ptr, delta_stride, delta_code = delta.data_ptr(), _matrix(delta, N, D, "delta"), _DTYPES[delta.dtype]
        if x_out is None:
            x_out = x
        if x_out.dtype != x_dtype:
            raise TypeError("x_out must have x's type")
        x_out_ptr, x_out_stride = x_out.data_ptr(), _matrix(x_out, N, D, "x_out")
    elif x_out is not None:
        raise ValueError("x_out without delta")
    if D == 0:
        raise ValueError("rows must not be empty")
    if out is None:
        out = rows_i8(N, D, x.device) if stream is None else _on(stream, rows_i8, N, D, x.device)
        q_stride = out.stride(0) if N > 1 else (D + 15) // 16 * 16
    else:
        q_stride = _bytes(out, N, D, "out")
    if scale is None:
        scale = torch.empty((N,), dtype=torch.float32, device=x.device) if stream is None else \
            _on(stream, torch.empty, (N,), dtype=torch.float32, device=x.device)
        scale_ptr = scale.data_ptr()
    else:
        scale_ptr = _scales(scale, N, "scale")
    if N:
        _enqueue(entry, index, stream, ROWS_ARGS.pack(
            out.data_ptr(), scale_ptr, x_out_ptr, x.data_ptr(), delta_ptr, weight_ptr, q_stride, x_stride, delta_stride, x_out_stride,
            N, D, eps, _DTYPES[x_dtype], delta_code))
    return out, scale


def rmsnorm_i8(x: torch.Tensor, weight: torch.Tensor, eps: float, *, delta=None, x_out=None, out=None, scale=None, stream=None):
    """(q, scale) of y = h / sqrt(mean(h^2) + eps) * weight, h = x + delta, per row: scale = max|y| / 127, q = round(y / scale).

    x       [N, D] fp32 / fp16 / bf16, rows may be strided; weight fp32 [D]; eps at least 2^-126
    delta   [N, D] of any of these types: the residual's addition. h is written to ``x_out`` (x's type; default: x itself)
    out     int8 [N, D] (rows_i8), scale fp32 [N]; new tensors by default
    A row of zeros has scale 0; one with NaN or an infinity q = 0 and scale NaN. Nothing that is written may share memory with
    another operand, but for x_out in the place of x."""
    return _rows("attn_rmsnorm_i8", x, weight, eps, delta, x_out, out, scale, stream)


def quantize_i8(x: torch.Tensor, *, out=None, scale=None, stream=None):
    """(q, scale) of the rows of x [N, D] fp32 / fp16 / bf16: scale = max|x| / 127, q = round(x / scale), ties to even. Of a weight
    matrix [n_out, k] the rows are the channels that gemm_i8 wants. Special rows and memory as rmsnorm_i8."""
    return _rows("attn_quantize_i8", x, None, 0.0, None, None, out, scale, stream)


def gemm_i8(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, *, out=None, out_dtype=torch.float32,
            swiglu: bool = False, status=None, stream=None) -> torch.Tensor:
    """out[t, j] = a_scale[t] * w_scale[j] * sum_i a[t, i] * w[j, i]: the sum exact, rounded once to out's type.

    a       int8 [m, k], a_scale fp32 [m]; w int8 [n, k], w_scale fp32 [n]; rows a multiple of 16 bytes apart, k up to 131071
    swiglu  w holds n_out gate rows, then n_out up rows: out = silu(gate) * up [m, n_out]
    out     fp32 / fp16 / bf16 [m, n_out], rows may be strided (default: a new tensor of out_dtype); no operand's memory
    The same bits for a token whatever else is in the batch."""
    index = _one_device(a, a_scale, w, w_scale, out, status)
    if a.dim() != 2 or w.dim() != 2:
        raise ValueError("a must be [m, k] and w [n, k]")
    m, k = a.shape
    w_rows = w.shape[0]
    if swiglu and w_rows % 2:
        raise ValueError("swiglu needs as many gate rows as up rows")
    n = w_rows // 2 if swiglu else w_rows
    a_stride, w_stride = _bytes(a, m, k, "a"), _bytes(w, w_rows, k, "w")
    a_scale_ptr, w_scale_ptr = _scales(a_scale, m, "a_scale"), _scales(w_scale, w_rows, "w_scale")
    if k > MAX_K or k == 0:
        raise ValueError(f"the inner dimension must be 1 to {MAX_K}")
    if out is None:
        ldc = 0
        out = torch.empty((m, n), dtype=out_dtype, device=a.device) if stream is None else \
            _on(stream, torch.empty, (m, n), dtype=out_dtype, device=a.device)
    else:
        ldc = _matrix(out, m, n, "out")
    if out.dtype not in _FLOATS:
        raise TypeError("out must be fp32, fp16 or bf16")
    if m and n:
        _enqueue("attn_gemm_i8", index, stream, GEMM_ARGS.pack(
            out.data_ptr(), a.data_ptr(), a_scale_ptr, w.data_ptr(), w_scale_ptr, a_stride, w_stride, ldc, m, n, k,
            _DTYPES[out.dtype], 1 if swiglu else 0, 0 if status is None else status.data_ptr()))
    return out
