"""Long contexts: scaled rotary positions, decode over a prefix that a batch shares, accumulated attention weights and eviction
from the caches. Torch tensors in, the C ABI underneath, in the manner of ``attention``.

The three belong to one generation path. ``rope_positions`` puts a token at any position into any cache row: behind a shared
prefix, or into a cache that evicted rows. ``attn_decode_shared`` attends the prefix and the own rows and adds up the weight each
own row received. ``kv_evict`` keeps the rows that matter when a cache is over its budget. ``model.Llama.generate_shared`` runs
them together.
"""
from __future__ import annotations

import math
import struct

import torch

from . import binding as _b
from .attention import _DTYPES, _dense, _dtype_code

_LAYOUTS = {"interleaved": _b.ROPE_INTERLEAVED, "half": _b.ROPE_HALF}
ROPE_LAYOUTS = tuple(sorted(_LAYOUTS))
_INDEX = (torch.int32, torch.uint32)
_CACHE = (torch.float16, torch.bfloat16)


def rope_frequencies(rotary_dim: int, theta: float, scaling: dict | None = None):
    """Radians per position of every pair (fp32, on the host) and the factor on cos and sin, for ``rope_positions``. ``scaling``
    is None or a dict with "type" and the fields its formula uses, under the names that model files give them:

    linear  factor                             every frequency / factor
    ntk     factor                             theta * factor ** (R / (R - 2)): the lowest frequency / factor, the highest kept
    yarn    factor, original (trained length), beta_fast = 32, beta_slow = 1, attention_factor = 0.1 ln(factor) + 1:
            frequencies that turn fewer than beta_slow times in the trained length / factor, more than beta_fast kept, a linear
            ramp over the pairs between
    llama3  factor, original, low_freq_factor = 1, high_freq_factor = 4: wavelengths longer than original / low_freq_factor
            / factor, shorter than original / high_freq_factor kept, a ramp over the turns between
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and positive")
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    freq = float(theta) ** (-2.0 * i / rotary_dim)
    if scaling is None:
        return freq.float(), 1.0
    kind, attention = scaling.get("type"), 1.0
    if kind not in ("linear", "ntk", "yarn", "llama3"):
        raise ValueError(f"unknown rotary scaling {kind!r}")
    factor = float(scaling["factor"])
    if not factor >= 1.0:
        raise ValueError("the scaling factor must be at least 1")
    if kind == "linear":
        freq = freq / factor
    elif kind == "ntk":
        if rotary_dim < 4:
            raise ValueError("ntk scaling needs at least two pairs")
        freq = (float(theta) * factor ** (rotary_dim / (rotary_dim - 2))) ** (-2.0 * i / rotary_dim)
    elif kind == "yarn":
        trained = float(scaling["original"])

        def pair_that_turns(n):
            return rotary_dim * math.log(trained / (n * 2 * math.pi)) / (2 * math.log(float(theta)))

        low = max(math.floor(pair_that_turns(scaling.get("beta_fast", 32.0))), 0)
        high = min(math.ceil(pair_that_turns(scaling.get("beta_slow", 1.0))), rotary_dim - 1)
        ramp = ((i - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        freq = freq / factor * ramp + freq * (1.0 - ramp)
        attention = float(scaling.get("attention_factor", 0.1 * math.log(factor) + 1.0))
    else:
        turns = float(scaling["original"]) * freq / (2 * math.pi)
        low, high = float(scaling.get("low_freq_factor", 1.0)), float(scaling.get("high_freq_factor", 4.0))
        if not high > low:
            raise ValueError("high_freq_factor must be larger than low_freq_factor")
        smooth = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        freq = (1.0 - smooth) * freq / factor + smooth * freq
    return freq.float(), attention


# The argument structures as the library lays them out. Packing one takes about a microsecond, filling the ctypes mirror field by
# field three, of the ten that a small call costs on the host.
ROPE_ARGS = struct.Struct("@10P6Q7If4iP")
SHARED_ARGS = struct.Struct("@7P2i6IPIf3Q2P2QPNP")
EVICT_ARGS = struct.Struct("@9P8I6QP")


def _enqueue(entry: str, index: int, stream, packed: bytes) -> None:
    """attention._call for a packed argument structure."""
    ptr = torch._C._cuda_getCurrentRawStream(index) if stream is None else stream.cuda_stream
    fn = getattr(_b.load(), entry)
    if torch._C._cuda_getDevice() == index:
        rc = fn(packed, ptr)
    else:
        with torch.cuda.device(index):
            rc = fn(packed, ptr)
    if rc:
        _b.check(rc, entry)


def _on(stream, make, *args, **kwargs):
    """What ``make`` allocates, for a kernel that runs on ``stream``: from that stream's memory, so that nothing the current stream
    still does, or does next, shares it."""
    with torch.cuda.stream(stream):
        return make(*args, **kwargs)


def _one_device(*tensors) -> int:
    """The index of the device that all operands are on."""
    index = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != index:
            index = -1
    if index < 0:
        raise ValueError("the operands must be CUDA tensors of one device (there is no CPU path)")
    return index


def _index(t, shape, what):
    if t.dtype not in _INDEX or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{what} must be a dense 32-bit integer CUDA tensor of shape {tuple(shape)}")
    return t.data_ptr()


def _score_stride(t: torch.Tensor, batch: int, kv_heads: int, rows: int) -> int:
    """Distance of the (sequence, kv head) runs of a [batch, kv_heads, rows] tensor of weights; 0 where there is one. (The library takes
    a distance of 0 as that of dense runs: an expanded tensor, whose runs are one, would be read and written behind its end.)"""
    stride = t.stride()
    apart = stride[1] if kv_heads > 1 else stride[0] if batch > 1 else rows
    if t.dtype != torch.float32 or t.shape != (batch, kv_heads, rows) or (rows > 1 and stride[2] != 1) or \
            (batch > 1 and kv_heads > 1 and stride[0] != kv_heads * stride[1]) or apart < rows:
        raise ValueError("scores must be fp32 [B, Hkv, rows] with dense rows at one distance, memory of their own each (not expanded)")
    return apart if kv_heads > 1 or batch > 1 else 0


def _row_stride(stride: int, rows: int, width: int, what: str) -> int:
    """Distance of the rows of a cache or prefix; 0, which the library takes as dense, where there is one."""
    if rows < 2:
        return 0
    if stride < width:
        raise ValueError(f"the rows of {what} must not share memory (expanded or overlapping rows)")
    return stride


def rope_positions(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   pos: torch.Tensor, row: torch.Tensor, *, inv_freq: torch.Tensor, seq=None, layout: str = "interleaved",
                   factor: float = 1.0, q_out=None, q_out_dtype=None, status=None, stream=None) -> torch.Tensor:
    """Rotates every token's q and k by ``pos * inv_freq`` and writes k and v into row ``row`` of sequence ``seq``'s caches.

    q [N, H, D], k / v [N, Hkv, D] fp32 / fp16 / bf16 (one type; views into a stacked projection are taken as they are);
    k_cache / v_cache fp16 / bf16 [B, T, Hkv, D]; pos, row, seq int32 CUDA tensors [N], not negative (seq None: token i is of sequence
    i); inv_freq fp32 [rotary_dim / 2] on the device and factor (0: 1) as rope_frequencies gives them, values behind rotary_dim are copied.
    layout "interleaved" pairs (2i, 2i + 1), "half" pairs (i, i + rotary_dim / 2). Returns the rotated q [N, H, D] (``q_out``, or a
    new tensor of q_out_dtype, default q's). A row that does not exist is not written and sets ATTN_STATUS_BAD_SHAPE in status."""
    index = _one_device(q, k, v, k_cache, v_cache, pos, row, inv_freq, seq, q_out, status)
    if q.dim() != 3 or k_cache.dim() != 4:
        raise ValueError("q must be [N, H, D], k and v [N, Hkv, D], the caches [B, T, Hkv, D]")
    N, H, D = q.shape
    B, T, Hkv, Dk = k_cache.shape
    if k.shape != (N, Hkv, D) or v.shape != (N, Hkv, D) or Dk != D or v_cache.shape != (B, T, Hkv, D):
        raise ValueError("shape mismatch between q, k, v and the caches")
    dtype, cache_dtype = q.dtype, k_cache.dtype
    if not (dtype == k.dtype == v.dtype) or cache_dtype not in _CACHE or v_cache.dtype != cache_dtype:
        raise TypeError("q, k, v must share a dtype, and the caches be both fp16 or both bf16")
    c_stride = k_cache.stride()
    if v_cache.stride() != c_stride or c_stride[3] != 1 or c_stride[2] != D:
        raise ValueError("the caches must be [B, row, kv_head, head_dim] with dense heads and share their strides")
    row_stride = _row_stride(c_stride[1], T, Hkv * D, "the caches")
    if layout not in _LAYOUTS:
        raise ValueError(f"layout must be one of {ROPE_LAYOUTS}")
    half = inv_freq.numel()
    if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or not inv_freq.is_contiguous() or not 0 < 2 * half <= D:
        raise ValueError("inv_freq must be a dense fp32 tensor of rotary_dim / 2 values, rotary_dim <= head_dim")
    if seq is None and N > B:
        raise ValueError("more tokens than sequences need seq")
    pos_ptr, row_ptr = _index(pos, (N,), "pos"), _index(row, (N,), "row")
    seq_ptr = 0 if seq is None else _index(seq, (N,), "seq")
    taken = []
    for t, what in ((q, "q"), (k, "k"), (v, "v")):
        stride = t.stride()
        if stride[2] != 1 or stride[1] != D or (N > 1 and stride[0] <= 0):
            t = _dense(t, stream, what)  # a token's heads must lie side by side; tokens may be strided
            stride = t.stride()
        taken += (t, stride[0] if N > 1 else 0)
    q, q_stride, k, k_stride, v, v_stride = taken
    out_stride = 0
    if q_out is None:
        o_dtype = q_out_dtype or dtype
        q_out = torch.empty_like(q, dtype=o_dtype, memory_format=torch.contiguous_format) if stream is None else \
            _on(stream, torch.empty_like, q, dtype=o_dtype, memory_format=torch.contiguous_format)
    else:
        stride = q_out.stride()
        if q_out.shape != (N, H, D) or stride[2] != 1 or stride[1] != D or (N > 1 and stride[0] < H * D):
            raise ValueError("q_out must be [N, H, D] with dense heads")
        out_stride = stride[0] if N > 1 else 0
    if N == 0:
        return q_out
    _enqueue("attn_rope_positions", index, stream, ROPE_ARGS.pack(
        q_out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), inv_freq.data_ptr(),
        pos_ptr, row_ptr, seq_ptr, q_stride, k_stride, v_stride, out_stride, row_stride, c_stride[0] if B > 1 else 0,
        N, H, Hkv, D, 2 * half, B, T, factor, _DTYPES[dtype], _dtype_code(q_out), _DTYPES[cache_dtype], _LAYOUTS[layout],
        0 if status is None else status.data_ptr()))
    return q_out


class SharedWorkspace:
    """Scratch of attn_decode_shared, reusable across calls of one shape on one stream; ``rows`` > 0 makes room for the scores
    of caches of that many rows."""

    def __init__(self, batch: int, n_heads: int, n_kv_heads: int, head_dim: int, rows: int = 0, device=None):
        device = torch.device("cuda" if device is None else device)
        if device.index is None:
            device = torch.device(device.type, torch.cuda.current_device())
        with torch.cuda.device(device):
            nbytes = _b.load().attn_decode_shared_workspace_bytes(batch, n_heads, n_kv_heads, head_dim, rows)
        if nbytes == 0:
            raise _b.AttnError(-2, f"no shared-prefix decode kernel for batch={batch} heads={n_heads}/{n_kv_heads} dim={head_dim}")
        self.key, self.rows = (batch, n_heads, n_kv_heads, head_dim, device.index), rows
        self.nbytes = int(nbytes)
        self.buf = torch.empty(self.nbytes, dtype=torch.uint8, device=device)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self.ptr, self.status_ptr = self.buf.data_ptr(), self.status.data_ptr()


def attn_decode_shared(q: torch.Tensor, k_prefix, v_prefix, k_cache: torch.Tensor, v_cache: torch.Tensor, kv_len=None, *,
                       out=None, lse=None, out_dtype=None, scale: float = 0.0, scores=None, scores_out=None,
                       workspace: SharedWorkspace | None = None, stream=None) -> torch.Tensor:
    """Single-token attention of a batch over a shared prefix and each sequence's own cache rows.

    q          [B, H, D]        fp16 / bf16, already rotated
    k_prefix   [P, Hkv, D]      q's type, or None (no prefix); rows may be strided. v_prefix the same
    k_cache    [B, T, Hkv, D]   q's type; rows and sequences may be strided (T may be 0). v_cache the same
    kv_len     None (all T rows), an int, or an int32 CUDA tensor [B] of valid own rows (0 is allowed)
    scores     [B, Hkv, T] fp32 accumulated weights, rows dense, each in memory of its own (not expanded); scores_out receives
               scores + this token's weights of the valid rows (default: scores itself, in place). scores_out alone starts from zero
    returns    out [B, H, D] in out_dtype (q's type, the default, or fp32); fills ``lse`` [B, H] (fp32) when given
    """
    index = _one_device(q, k_prefix, v_prefix, k_cache, v_cache, kv_len if isinstance(kv_len, torch.Tensor) else None, out, lse, scores,
                        scores_out)
    if q.dim() != 3 or k_cache.dim() != 4:
        raise ValueError("q must be [B, H, D] and the caches [B, T, Hkv, D]")
    B, H, D = q.shape
    Bk, T, Hkv, Dk = k_cache.shape
    if Bk != B or Dk != D or v_cache.shape != (B, T, Hkv, D) or Hkv == 0 or H % Hkv:
        raise ValueError("shape mismatch between q and the caches")
    dtype = q.dtype
    if dtype not in _CACHE or k_cache.dtype != dtype or v_cache.dtype != dtype:
        raise TypeError("q and the caches must be fp16 or bf16, of one type")
    stride = k_cache.stride()
    if v_cache.stride() != stride or (T and (stride[3] != 1 or stride[2] != D)):
        raise ValueError("the caches must be [B, row, kv_head, head_dim] with dense heads and share their strides")
    row_stride = _row_stride(stride[1], T, Hkv * D, "the caches")
    P = kp = vp = prefix_stride = 0
    if (k_prefix is None) != (v_prefix is None):
        raise ValueError("k_prefix without v_prefix")
    if k_prefix is not None:
        P, Hp, Dp = k_prefix.shape if k_prefix.dim() == 3 else (0, 0, 0)
        if Hp != Hkv or Dp != D or v_prefix.shape != k_prefix.shape:
            raise ValueError("the prefix must be [P, Hkv, D]")
        if k_prefix.dtype != dtype or v_prefix.dtype != dtype:
            raise TypeError("the prefix must have q's type")
        if P:
            p_stride = k_prefix.stride()
            if v_prefix.stride() != p_stride or p_stride[2] != 1 or p_stride[1] != D:
                raise ValueError("the prefix must be [row, kv_head, head_dim] with dense heads; K and V share their strides")
            kp, vp, prefix_stride = k_prefix.data_ptr(), v_prefix.data_ptr(), _row_stride(p_stride[0], P, Hkv * D, "the prefix")
    len_ptr, uniform = 0, T
    if isinstance(kv_len, int):
        if not 0 <= kv_len <= T:
            raise ValueError("kv_len exceeds the cache")
        uniform = kv_len
    elif kv_len is not None:
        len_ptr = _index(kv_len, (B,), "kv_len")
    if scores is not None and scores_out is None:
        scores_out = scores
    scores_ptr = scores_out_ptr = score_stride = score_out_stride = 0
    if scores_out is not None:
        score_out_stride = _score_stride(scores_out, B, Hkv, T)
        if scores is not None:
            score_stride = _score_stride(scores, B, Hkv, T)
        if T:  # (without rows there is nothing to add up)
            scores_out_ptr, scores_ptr = scores_out.data_ptr(), 0 if scores is None else scores.data_ptr()
    if not q.is_contiguous():
        q = _dense(q, stream, "q")
    if out is None:
        o_dtype = out_dtype or dtype  # (q is dense: empty_like, which takes half the host time of torch.empty)
        out = torch.empty_like(q, dtype=o_dtype) if stream is None else _on(stream, torch.empty_like, q, dtype=o_dtype)
    elif out.shape != (B, H, D) or not out.is_contiguous():
        raise ValueError("out must be a contiguous [B, H, D] tensor")
    o_dtype = out.dtype
    if o_dtype != dtype and o_dtype != torch.float32:
        raise TypeError("out must have q's type or be fp32")
    if lse is not None and (lse.dtype != torch.float32 or lse.shape != (B, H) or not lse.is_contiguous()):
        raise ValueError("lse must be a contiguous fp32 [B, H] tensor")
    if B == 0:
        return out
    need_rows = T if scores_out_ptr else 0
    if workspace is None or workspace.key != (B, H, Hkv, D, index) or workspace.rows < need_rows:
        shape = (B, H, Hkv, D, need_rows, q.device)
        workspace = SharedWorkspace(*shape) if stream is None else _on(stream, SharedWorkspace, *shape)
    _enqueue("attn_decode_shared", index, stream, SHARED_ARGS.pack(
        out.data_ptr(), q.data_ptr(), kp, vp, k_cache.data_ptr() if T else 0, v_cache.data_ptr() if T else 0,
        0 if lse is None else lse.data_ptr(), _DTYPES[o_dtype], _DTYPES[dtype], B, H, Hkv, D, P, T, len_ptr, uniform,
        scale, prefix_stride, row_stride, stride[0] if B > 1 else 0, scores_ptr, scores_out_ptr, score_stride,
        score_out_stride, workspace.ptr, workspace.nbytes, workspace.status_ptr))
    return out


def kv_evict(k_cache: torch.Tensor, v_cache: torch.Tensor, scores: torch.Tensor, kv_len, keep: int, *, sink: int = 0,
             recent: int = 0, out=None, kept=None, kv_len_out=None, status=None, stream=None):
    """Keeps, per sequence and kv head, the first ``sink`` rows, the last ``recent`` rows and those with the largest scores up to
    ``keep`` rows, in their order.

    k_cache, v_cache [B, T, Hkv, D] 16-bit, scores [B, Hkv, T] fp32 with dense rows, kv_len an int32 CUDA tensor [B] or None (T).
    out  None: in place; or (k_out, v_out, scores_out) with [B, T2, Hkv, D] and [B, Hkv, T2], T2 >= keep, sharing no byte with
         the inputs or each other. K and V rows behind a new length are left alone, scores there become 0.
    Returns (kept [B, Hkv, keep] int32: the source row of each kept row, -1 behind the new length; kv_len_out [B] int32:
    min(length, keep); it may be given as kv_len itself)."""
    k_out, v_out, scores_out = (k_cache, v_cache, scores) if out is None else out
    index = _one_device(k_cache, v_cache, scores, k_out, v_out, scores_out, kv_len, kept, kv_len_out, status)
    if k_cache.dim() != 4 or k_out.dim() != 4:
        raise ValueError("the caches must be [B, T, Hkv, D]")
    B, T, Hkv, D = k_cache.shape
    T2 = k_out.shape[1]
    dtype = k_cache.dtype
    s_in, s_out = k_cache.stride(), k_out.stride()
    if v_cache.shape != k_cache.shape or k_out.shape != (B, T2, Hkv, D) or v_out.shape != k_out.shape or v_cache.stride() != s_in or \
            v_out.stride() != s_out or s_in[3] != 1 or s_in[2] != D or s_out[3] != 1 or s_out[2] != D:
        raise ValueError("the caches must be [B, row, kv_head, head_dim] with dense heads; K and V share their strides")
    if dtype not in _CACHE or not (v_cache.dtype == k_out.dtype == v_out.dtype == dtype):
        raise TypeError("the caches must be fp16 or bf16, of one type")
    row_in, row_out = _row_stride(s_in[1], T, Hkv * D, "the caches"), _row_stride(s_out[1], T2, Hkv * D, "the output caches")
    score_stride, score_out_stride = _score_stride(scores, B, Hkv, T), _score_stride(scores_out, B, Hkv, T2)
    if keep < 1 or keep > T2 or sink < 0 or recent < 0 or sink + recent > keep:
        raise ValueError("keep must be at least 1, fit the output caches and hold the sink and the recent rows")
    if kept is None:
        shape, stride, device = (B, Hkv, keep), (Hkv * keep, keep, 1), k_cache.device
        kept = torch.empty_strided(shape, stride, dtype=torch.int32, device=device) if stream is None else \
            _on(stream, torch.empty_strided, shape, stride, dtype=torch.int32, device=device)
        kept_ptr = kept.data_ptr()
    else:
        kept_ptr = _index(kept, (B, Hkv, keep), "kept")
    len_ptr = 0 if kv_len is None else _index(kv_len, (B,), "kv_len")
    if kv_len_out is None:
        if stream is not None:
            kv_len_out = _on(stream, torch.empty, (B,), dtype=torch.int32, device=k_cache.device)
        else:
            kv_len_out = torch.empty((B,), dtype=torch.int32, device=k_cache.device) if kv_len is None else torch.empty_like(kv_len)
        len_out_ptr = kv_len_out.data_ptr()
    else:
        len_out_ptr = _index(kv_len_out, (B,), "kv_len_out")
    if B == 0:
        return kept, kv_len_out
    _enqueue("attn_kv_evict", index, stream, EVICT_ARGS.pack(
        k_cache.data_ptr(), v_cache.data_ptr(), k_out.data_ptr(), v_out.data_ptr(), scores.data_ptr(), scores_out.data_ptr(), kept_ptr,
        len_ptr, len_out_ptr, B, Hkv, D, T, T2, keep, sink, recent,
        row_in, row_out, s_in[0] if B > 1 else 0, s_out[0] if B > 1 else 0, score_stride,
        score_out_stride, 0 if status is None else status.data_ptr()))
    return kept, kv_len_out
