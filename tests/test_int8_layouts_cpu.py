"""What the 8-bit integer operators make of their operands' layouts, without a device: tensors of the host stand in, and what would be
handed to the library is looked at instead."""
import types

import pytest
import torch


@pytest.fixture
def i8(built_lib, pkg, monkeypatch):
    from llm_infer_b200 import int8
    calls = []
    monkeypatch.setattr(int8, "_one_device", lambda *tensors: 0)
    monkeypatch.setattr(int8, "_enqueue", lambda entry, index, stream, packed: calls.append((entry, packed)))
    return types.SimpleNamespace(op=int8, calls=calls, b=pkg.binding)


def _last(i8):
    entry, packed = i8.calls[-1]
    mirror = i8.b.AttnGemmI8Args if entry == "attn_gemm_i8" else i8.b.AttnRowsI8Args
    return mirror.from_buffer_copy(packed)


def test_strides_of_rows(i8):
    big = torch.zeros((6, 100))
    w = torch.ones(40)
    for x, delta, x_out, strides in (
            (torch.zeros((5, 40)), torch.zeros((5, 40)).half(), torch.zeros((5, 40)), (0, 0, 0)),
            (big[:5, :40], big[1:, 40:80], torch.zeros((5, 50))[:, 10:], (100, 100, 50)),
            (big[:1, :40], big[1:2, 40:80], torch.zeros((5, 40))[:1], (0, 0, 0)),
            (torch.zeros((40, 5)).t()[:1].contiguous(), None, None, (0, 0, 0))):
        if x.shape[1] != 40:
            continue
        q, s = i8.op.rmsnorm_i8(x, w, 1e-5, delta=delta, x_out=x_out)
        a = _last(i8)
        assert (a.x_stride, a.delta_stride, a.x_out_stride) == strides and (a.rows, a.dim) == x.shape
        assert a.x == x.data_ptr() and a.q == q.data_ptr() and a.scale == s.data_ptr() and a.weight == w.data_ptr()
        assert a.delta == (0 if delta is None else delta.data_ptr()) or a.delta is None
        assert a.q_stride == 48


def test_x_out_is_x_where_none_is_given(i8):
    x, d = torch.zeros((5, 40)).bfloat16(), torch.zeros((5, 40))
    i8.op.rmsnorm_i8(x, torch.ones(40), 1e-5, delta=d)
    a = _last(i8)
    assert a.x_out == a.x == x.data_ptr() and (a.x_dtype, a.delta_dtype) == (i8.b.DTYPE_BF16, i8.b.DTYPE_F32)
    i8.op.quantize_i8(x)
    a = _last(i8)
    assert a.x_out is None and a.delta is None and a.weight is None


def test_strides_of_products(i8):
    one = torch.ones(7)
    for q, stride in ((i8.op.rows_i8(7, 40, "cpu"), 48), (i8.op.rows_i8(7, 160, "cpu"), 256), (torch.zeros((7, 160), dtype=torch.int8), 0),
                      (torch.zeros((7, 400), dtype=torch.int8)[:, 16:56], 400), (torch.zeros((7, 40), dtype=torch.int8)[:1], 0)):
        m, k = q.shape
        out = i8.op.gemm_i8(q, one[:m], q, one[:m], out=torch.zeros((m, 20))[:, 3:3 + m], w_early=True)
        a = _last(i8)
        assert (a.a_stride, a.w_stride) == (stride, stride) and (a.m, a.n_out, a.k) == (m, m, k)
        assert a.ldc == (20 if m > 1 else 0) and a.out == out.data_ptr() and a.w_early == 1 and a.swiglu == 0
    w = torch.zeros((14, 160), dtype=torch.int8)
    out = i8.op.gemm_i8(torch.zeros((3, 160), dtype=torch.int8), one[:3], w, torch.ones(14), swiglu=True, out_dtype=torch.float16)
    a = _last(i8)
    assert out.shape == (3, 7) and a.n_out == 7 and a.swiglu == 1 and a.out_dtype == i8.b.DTYPE_F16 and a.ldc == 0


@pytest.mark.parametrize("make", [lambda: torch.zeros((1, 160), dtype=torch.int8).expand(7, 160),
                                  lambda: torch.zeros(2000, dtype=torch.int8).as_strided((7, 160), (144, 1)),
                                  lambda: torch.zeros((160, 7), dtype=torch.int8).t(),
                                  lambda: torch.zeros((7, 200), dtype=torch.int8)[:, :160],
                                  lambda: torch.zeros((7, 320), dtype=torch.int8)[:, ::2]],
                         ids=["expanded", "overlapping", "transposed", "200 bytes apart", "every second byte"])
def test_rows_that_share_memory_or_lie_oddly_are_refused(i8, make):
    one, good = torch.ones(7), torch.zeros((7, 160), dtype=torch.int8)
    for call in (lambda: i8.op.gemm_i8(make(), one, good, one), lambda: i8.op.gemm_i8(good, one, make(), one),
                 lambda: i8.op.quantize_i8(torch.zeros((7, 160)), out=make())):
        with pytest.raises(ValueError, match="rows"):
            call()
    assert not i8.calls


@pytest.mark.parametrize("make", [lambda: torch.zeros((1, 40)).expand(7, 40), lambda: torch.zeros(300).as_strided((7, 40), (39, 1)),
                                  lambda: torch.zeros((40, 7)).t(), lambda: torch.zeros((7, 80))[:, ::2]],
                         ids=["expanded", "overlapping", "transposed", "every second value"])
def test_floating_rows_that_share_memory_or_lie_oddly_are_refused(i8, make):
    good, w = torch.zeros((7, 40)), torch.ones(40)
    for call in (lambda: i8.op.quantize_i8(make()), lambda: i8.op.rmsnorm_i8(make(), w, 1e-5), lambda: i8.op.rmsnorm_i8(good, w, 1e-5, delta=make()),
                 lambda: i8.op.rmsnorm_i8(good, w, 1e-5, delta=good.clone(), x_out=make()),
                 lambda: i8.op.gemm_i8(torch.zeros((7, 16), dtype=torch.int8), torch.ones(7), torch.zeros((40, 16), dtype=torch.int8), torch.ones(40),
                                       out=make())):
        with pytest.raises(ValueError, match="rows"):
            call()
    assert not i8.calls


def test_scales_that_are_not_dense_are_refused(i8):
    q = torch.zeros((7, 160), dtype=torch.int8)
    for bad in (torch.ones(8), torch.ones(14)[::2], torch.ones(1).expand(7), torch.ones((7, 1)), torch.ones(7).half()):
        for call in (lambda: i8.op.gemm_i8(q, bad, q, torch.ones(7)), lambda: i8.op.gemm_i8(q, torch.ones(7), q, bad),
                     lambda: i8.op.quantize_i8(torch.zeros((7, 40)), scale=bad)):
            with pytest.raises(ValueError, match="scale"):
                call()
    assert not i8.calls
