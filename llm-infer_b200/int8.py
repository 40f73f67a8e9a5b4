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
from .context import _INDEX, _enqueue, _on, _one_device

_F32, _I8 = torch.float32, torch.int8
_FLOATS = {t: _DTYPES[t] for t in (torch.float32, torch.float16, torch.bfloat16)}
MAX_K = 131071  # longest inner dimension of gemm_i8: 32-bit sums of products of 8 bits stay exact

# The argument structures as the library lays them out (packed: see context).
ROWS_ARGS = struct.Struct("@6P4Q2If2iP")
GEMM_ARGS = struct.Struct("@5P3Q3I2iPi0P")


def rows_i8(rows: int, k: int, device=None) -> torch.Tensor:
    """An int8 tensor [rows, k] laid out as the operators take it: rows a multiple of 16 bytes apart, from k = 128 on a multiple of 128,
    which is what memory is read in (10525 x 2948 x 2048: 64.6 us with rows 2960 bytes apart, 51.1 so)."""
    return torch.empty_strided((rows, k), (_apart(k), 1), dtype=_I8, device="cuda" if device is None else device)


def _apart(k: int) -> int:
    return (k + 127) & ~127 if k >= 128 else (k + 15) & ~15


# (A call's checks are part of the microseconds that a small one takes: what is dense is asked first, the rest is looked at here.)
def _row_stride(t: torch.Tensor, rows: int, dim: int, what: str) -> int:
    """Distance of the rows of a [rows, dim] tensor; 0, which the library takes as dense, where there is one."""
    stride = t.stride()
    if dim > 1 and stride[1] != 1:
        raise ValueError(f"the rows of {what} must be dense")
    if rows < 2:
        return 0
    if stride[0] < dim:
        raise ValueError(f"the rows of {what} must not share memory (expanded or overlapping rows)")
    return stride[0]


def _byte_stride(q: torch.Tensor, rows: int, k: int, what: str) -> int:
    """The same for an 8-bit matrix, whose rows are a multiple of 16 bytes apart (0: k rounded up to one)."""
    stride = _row_stride(q, rows, k, what)
    if stride % 16:
        raise ValueError(f"the rows of {what} must be a multiple of 16 bytes apart (rows_i8 lays them out so)")
    return stride


def _status(t: torch.Tensor) -> int:
    """The address of a status word."""
    if t.dtype not in _INDEX or t.numel() == 0:
        raise ValueError("status must be a tensor of 32-bit integers, its first element the word")
    return t.data_ptr()


def _rows(entry: str, x, weight, eps: float, delta, x_out, out, scale, status, stream):
    index = _one_device(x, weight, delta, x_out, out, scale, status)
    shape, x_dtype = x.shape, x.dtype
    if len(shape) != 2 or shape[1] == 0:
        raise ValueError("x must be [N, D], its rows not empty")
    N, D = shape
    x_code = _FLOATS.get(x_dtype)
    if x_code is None:
        raise TypeError("x must be fp32, fp16 or bf16")
    x_stride = 0 if x.is_contiguous() else _row_stride(x, N, D, "x")
    weight_ptr = delta_ptr = delta_stride = delta_code = x_out_ptr = x_out_stride = 0
    if weight is not None:
        if weight.dtype is not _F32 or weight.shape != (D,) or not weight.is_contiguous():
            raise ValueError(f"weight must be a dense fp32 tensor [{D}]")
        weight_ptr = weight.data_ptr()
    if delta is not None:
        delta_code = _FLOATS.get(delta.dtype)
        if delta_code is None:
            raise TypeError("delta must be fp32, fp16 or bf16")
        if x_out is None:
            x_out = x
        if delta.shape != shape or x_out.shape != shape or x_out.dtype != x_dtype:
            raise ValueError("delta and x_out must have x's shape, x_out its type")
        delta_ptr, delta_stride = delta.data_ptr(), 0 if delta.is_contiguous() else _row_stride(delta, N, D, "delta")
        x_out_ptr, x_out_stride = x_out.data_ptr(), 0 if x_out.is_contiguous() else _row_stride(x_out, N, D, "x_out")
    elif x_out is not None:
        raise ValueError("x_out without delta")
    if out is None:
        out = rows_i8(N, D, x.device) if stream is None else _on(stream, rows_i8, N, D, x.device)
        q_stride = _apart(D)
    else:
        if out.dtype is not _I8 or out.shape != shape:
            raise ValueError("out must be int8, of x's shape")
        q_stride = _byte_stride(out, N, D, "out")
    if scale is None:
        scale = torch.empty_strided((N,), (1,), dtype=torch.float32, device=x.device) if stream is None else \
            _on(stream, torch.empty_strided, (N,), (1,), dtype=torch.float32, device=x.device)
    elif scale.dtype is not _F32 or scale.shape != (N,) or not scale.is_contiguous():
        raise ValueError(f"scale must be a dense fp32 tensor [{N}]")
    if N:
        _enqueue(entry, index, stream, ROWS_ARGS.pack(
            out.data_ptr(), scale.data_ptr(), x_out_ptr, x.data_ptr(), delta_ptr, weight_ptr, q_stride, x_stride, delta_stride,
            x_out_stride, N, D, eps, x_code, delta_code, 0 if status is None else _status(status)))
    return out, scale


def rmsnorm_i8(x: torch.Tensor, weight: torch.Tensor, eps: float, *, delta=None, x_out=None, out=None, scale=None, status=None,
               stream=None):
    """(q, scale) of y = h / sqrt(mean(h^2) + eps) * weight, h = x + delta, per row: scale = max|y| / 127, q = round(y / scale).

    x       [N, D] fp32 / fp16 / bf16, rows may be strided; weight fp32 [D]; eps at least 2^-126
    delta   [N, D] of any of these types: the residual's addition. h is written to ``x_out`` (x's type; default: x itself)
    out     int8 [N, D] (rows_i8), scale fp32 [N]; new tensors by default
    status  optional device word for ATTN_STATUS_* bits: rows that did not arrive have q = 0 and scale NaN, and x_out is not written, or in part
    A row of zeros has scale 0; one with NaN or an infinity, or whose h * weight or sum of h^2 passes fp32's range (|h| of 1.8e19 / sqrt(D)
    throughout), q = 0 and scale NaN. Nothing that is written may share memory with another operand, but for x_out in the place of x;
    rows between another operand's rows, at the same distance, share none."""
    return _rows("attn_rmsnorm_i8", x, weight, eps, delta, x_out, out, scale, status, stream)


def quantize_i8(x: torch.Tensor, *, out=None, scale=None, status=None, stream=None):
    """(q, scale) of the rows of x [N, D] fp32 / fp16 / bf16: scale = max|x| / 127, q = round(x / scale), ties to even. Of a weight
    matrix [n_out, k] the rows are the channels that gemm_i8 wants. Special rows and memory as rmsnorm_i8."""
    return _rows("attn_quantize_i8", x, None, 0.0, None, None, out, scale, status, stream)


def gemm_i8(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, *, out=None, out_dtype=torch.float32,
            swiglu: bool = False, status=None, w_early: bool = False, stream=None) -> torch.Tensor:
    """out[t, j] = a_scale[t] * w_scale[j] * sum_i a[t, i] * w[j, i]: the sum exact in 32-bit integers, then converted to
    fp32 (rounded beyond 2^24), times w_scale[j], times a_scale[t], each rounded to fp32, and rounded to out's type.

    a       int8 [m, k], a_scale fp32 [m]; w int8 [n, k], w_scale fp32 [n]; rows a multiple of 16 bytes apart, k up to 131071
    swiglu  w holds n_out gate rows, then n_out up rows: out = silu(gate) * up [m, n_out]
    out     fp32 / fp16 / bf16 [m, n_out], rows may be strided (default: a new tensor of out_dtype); no operand's memory
    w_early the caller vouches that what wrote w had completed, the host having waited for it (torch.cuda.synchronize), before the
            previous kernel of the stream was enqueued, as for a loaded model's weights: its first tiles are then read while that kernel,
            and those in front of it, may still be running. A quantize_i8 of w further ahead in the stream is not waited for
    The same bits for a token whatever else is in the batch."""
    index = _one_device(a, a_scale, w, w_scale, out, status)
    a_shape, w_shape = a.shape, w.shape
    if len(a_shape) != 2 or len(w_shape) != 2 or a_shape[1] != w_shape[1]:
        raise ValueError("a must be [m, k] and w [n, k]")
    m, k = a_shape
    n = rows = w_shape[0]
    if not 0 < k <= MAX_K:
        raise ValueError(f"the inner dimension must be 1 to {MAX_K}")
    if swiglu:
        if rows % 2:
            raise ValueError("swiglu needs as many gate rows as up rows")
        n //= 2
    if a.dtype is not _I8 or w.dtype is not _I8:
        raise TypeError("a and w must be int8")
    packed = k % 16 == 0
    a_stride = 0 if packed and a.is_contiguous() else _byte_stride(a, m, k, "a")
    w_stride = 0 if packed and w.is_contiguous() else _byte_stride(w, rows, k, "w")
    if a_scale.dtype is not _F32 or w_scale.dtype is not _F32 or a_scale.shape != (m,) or w_scale.shape != (rows,) or \
            not (a_scale.is_contiguous() and w_scale.is_contiguous()):
        raise ValueError(f"a_scale and w_scale must be dense fp32 tensors [{m}] and [{rows}]")
    ldc = 0
    if out is None:
        out = torch.empty_strided((m, n), (n, 1), dtype=out_dtype, device=a.device) if stream is None else \
            _on(stream, torch.empty_strided, (m, n), (n, 1), dtype=out_dtype, device=a.device)
    else:
        if out.shape != (m, n):
            raise ValueError(f"out must be [{m}, {n}]")
        if not out.is_contiguous():
            ldc = _row_stride(out, m, n, "out")
    out_code = _FLOATS.get(out.dtype)
    if out_code is None:
        raise TypeError("out must be fp32, fp16 or bf16")
    if m and n:
        _enqueue("attn_gemm_i8", index, stream, GEMM_ARGS.pack(
            out.data_ptr(), a.data_ptr(), a_scale.data_ptr(), w.data_ptr(), w_scale.data_ptr(), a_stride, w_stride, ldc, m, n, k,
            out_code, 1 if swiglu else 0, 0 if status is None else _status(status), 1 if w_early else 0))
    return out
