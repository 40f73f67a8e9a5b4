"""8-bit integer operators without a device: what they refuse, and the layout of their arguments."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def i8(built_lib, pkg):
    from llm_infer_b200 import int8
    return int8


def _rows_args(b):
    a = b.AttnRowsI8Args()
    for i, n in enumerate("q scale x_out x delta weight".split()):
        setattr(a, n, (i + 1) << 20)
    a.rows, a.dim, a.eps = 5, 100, 1e-5
    a.x_dtype, a.delta_dtype = b.DTYPE_F32, b.DTYPE_F16
    return a


def _plain_args(b):
    a = _rows_args(b)
    a.x_out = a.delta = a.weight = None
    return a


def _gemm_args(b):
    a = b.AttnGemmI8Args()
    for i, n in enumerate("out a a_scale w w_scale".split()):
        setattr(a, n, (i + 1) << 24)
    a.m, a.n_out, a.k = 5, 100, 70
    return a


@pytest.mark.parametrize("entry,make,changes,code", [
    ("attn_rmsnorm_i8", _rows_args, dict(q=None), -1),
    ("attn_rmsnorm_i8", _rows_args, dict(scale=None), -1),
    ("attn_rmsnorm_i8", _rows_args, dict(x=None), -1),
    ("attn_rmsnorm_i8", _rows_args, dict(weight=None), -1),
    ("attn_rmsnorm_i8", _rows_args, dict(rows=0), -1),
    ("attn_rmsnorm_i8", _rows_args, dict(dim=0), -1),
    ("attn_rmsnorm_i8", _rows_args, dict(eps=0.0), -1),
    ("attn_rmsnorm_i8", _rows_args, dict(eps=-1e-5), -1),
    ("attn_rmsnorm_i8", _rows_args, dict(eps=float("nan")), -1),
    ("attn_rmsnorm_i8", _rows_args, dict(eps=float("inf")), -1),
    ("attn_rmsnorm_i8", _rows_args, dict(eps=1e-39), -1),                 # below fp32's normal numbers
    ("attn_rmsnorm_i8", _rows_args, dict(x_dtype=3), -1),
    ("attn_rmsnorm_i8", _rows_args, dict(delta_dtype=4), -1),
    ("attn_rmsnorm_i8", _rows_args, dict(delta=None), -1),                # x_out without delta
    ("attn_rmsnorm_i8", _rows_args, dict(rows=1 << 31), -2),
    ("attn_rmsnorm_i8", _rows_args, dict(q_stride=96), -1),               # rows would overlap
    ("attn_rmsnorm_i8", _rows_args, dict(x_stride=99), -1),
    ("attn_rmsnorm_i8", _rows_args, dict(delta_stride=99), -1),
    ("attn_rmsnorm_i8", _rows_args, dict(x_out_stride=99), -1),
    ("attn_rmsnorm_i8", _rows_args, dict(q_stride=104), -3),
    ("attn_rmsnorm_i8", _rows_args, dict(q=(1 << 20) + 8), -3),
    ("attn_rmsnorm_i8", _rows_args, dict(x=(4 << 20) + 2), -3),
    ("attn_rmsnorm_i8", _rows_args, dict(delta=(5 << 20) + 1), -3),
    ("attn_rmsnorm_i8", _rows_args, dict(weight=(6 << 20) + 2), -3),
    ("attn_rmsnorm_i8", _rows_args, dict(scale=(2 << 20) + 2), -3),
    ("attn_rmsnorm_i8", _rows_args, dict(x_out=(4 << 20) + 400), -1),     # a row further on in x
    ("attn_rmsnorm_i8", _rows_args, dict(x_out=4 << 20, x_out_stride=200), -1),
    ("attn_rmsnorm_i8", _rows_args, dict(x_out=5 << 20), -1),             # the delta's memory
    ("attn_rmsnorm_i8", _rows_args, dict(x_out=6 << 20), -1),             # the weight's
    ("attn_rmsnorm_i8", _rows_args, dict(q=4 << 20), -1),
    ("attn_rmsnorm_i8", _rows_args, dict(q=5 << 20), -1),
    ("attn_rmsnorm_i8", _rows_args, dict(scale=(4 << 20) + 1996), -1),    # the last value of x
    ("attn_rmsnorm_i8", _rows_args, dict(scale=1 << 20), -1),
    ("attn_rmsnorm_i8", _rows_args, dict(scale=(6 << 20) + 396), -1),
    ("attn_quantize_i8", _plain_args, dict(weight=1 << 24), -1),
    ("attn_quantize_i8", _plain_args, dict(delta=1 << 24), -1),
    ("attn_quantize_i8", _plain_args, dict(x_out=1 << 24), -1),
    ("attn_quantize_i8", _plain_args, dict(x=None), -1),
    ("attn_quantize_i8", _plain_args, dict(q=4 << 20), -1),
    ("attn_gemm_i8", _gemm_args, dict(out=None), -1),
    ("attn_gemm_i8", _gemm_args, dict(a=None), -1),
    ("attn_gemm_i8", _gemm_args, dict(a_scale=None), -1),
    ("attn_gemm_i8", _gemm_args, dict(w=None), -1),
    ("attn_gemm_i8", _gemm_args, dict(w_scale=None), -1),
    ("attn_gemm_i8", _gemm_args, dict(m=0), -1),
    ("attn_gemm_i8", _gemm_args, dict(n_out=0), -1),
    ("attn_gemm_i8", _gemm_args, dict(k=0), -1),
    ("attn_gemm_i8", _gemm_args, dict(k=131072), -2),                     # sums could pass 32 bits
    ("attn_gemm_i8", _gemm_args, dict(out_dtype=3), -1),
    ("attn_gemm_i8", _gemm_args, dict(ldc=99), -1),
    ("attn_gemm_i8", _gemm_args, dict(a_stride=64), -1),
    ("attn_gemm_i8", _gemm_args, dict(w_stride=64), -1),
    ("attn_gemm_i8", _gemm_args, dict(a_stride=72), -3),
    ("attn_gemm_i8", _gemm_args, dict(w_stride=88), -3),
    ("attn_gemm_i8", _gemm_args, dict(a=(2 << 24) + 4), -3),
    ("attn_gemm_i8", _gemm_args, dict(w=(4 << 24) + 8), -3),
    ("attn_gemm_i8", _gemm_args, dict(out=(1 << 24) + 2), -3),
    ("attn_gemm_i8", _gemm_args, dict(out=2 << 24), -1),                  # over a
    ("attn_gemm_i8", _gemm_args, dict(out=(4 << 24) - 1600), -1),         # its end over w
    ("attn_gemm_i8", _gemm_args, dict(out=5 << 24), -1),
    ("attn_gemm_i8", _gemm_args, dict(out=3 << 24), -1),
])
def test_bad_arguments_are_refused_before_a_device_is_touched(built_lib, pkg, entry, make, changes, code):
    a = make(pkg.binding)
    for name, value in changes.items():
        setattr(a, name, value)
    assert getattr(built_lib, entry)(C.byref(a), None) == code
    assert getattr(built_lib, entry)(None, None) == -1


def test_operands_beside_each_other_are_not_refused_as_shared(built_lib, pkg):
    """Columns of one buffer: x, delta and x_out side by side, and out between the rows of nothing it shares a byte with. Without a
    device such a call gets as far as asking for one."""
    a = _rows_args(pkg.binding)
    a.x, a.x_out, a.x_stride, a.x_out_stride = 4 << 20, (4 << 20) + 400, 200, 200
    if not torch.cuda.is_available():
        assert built_lib.attn_rmsnorm_i8(C.byref(a), None) == -5


def test_packed_arguments_lie_as_the_structures_do(i8, pkg):
    b = pkg.binding
    for packed, mirror in ((i8.ROWS_ARGS, b.AttnRowsI8Args), (i8.GEMM_ARGS, b.AttnGemmI8Args)):
        assert packed.size == C.sizeof(mirror)
        names = [n for n, _ in mirror._fields_]
        values = [float(i + 1) if t is C.c_float else i + 1 for i, (_, t) in enumerate(mirror._fields_)]
        a = mirror.from_buffer_copy(packed.pack(*values))
        assert [getattr(a, n) for n in names] == values


def test_cpu_tensors_are_refused(i8):
    x, w = torch.zeros(3, 32), torch.ones(32)
    q, s = torch.zeros((3, 32), dtype=torch.int8), torch.zeros(3)
    for call in (lambda: i8.rmsnorm_i8(x, w, 1e-5), lambda: i8.quantize_i8(x), lambda: i8.gemm_i8(q, s, q, s)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_rows_are_a_multiple_of_sixteen_bytes_apart(i8):
    for k, apart in ((1, 16), (15, 16), (16, 16), (17, 32), (127, 128), (128, 128), (129, 256), (4096, 4096), (5003, 5120)):
        q = i8.rows_i8(3, k, "cpu")
        assert q.shape == (3, k) and q.stride() == (apart, 1) and q.dtype == torch.int8
