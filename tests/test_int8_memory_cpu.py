"""Which operands the 8-bit entry points take for sharing memory, asked without a device: a call that is not refused gets as far as
looking for one."""
import ctypes as C

import pytest
import torch

from test_int8_cpu import _gemm_args, _rows_args

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are made up: a device would be handed them")
NO_DEVICE, REFUSED = -5, -1
B = 1 << 24


def _call(lib, entry, args, **changes):
    for name, value in changes.items():
        setattr(args, name, value)
    return getattr(lib, entry)(C.byref(args), None)


@pytest.mark.parametrize("changes,code", [
    (dict(x=B, delta=B + 400, x_out=B + 800, q=B + 1200, x_stride=400, delta_stride=800, x_out_stride=400, q_stride=1600), NO_DEVICE),
    (dict(x=B, delta=B + 400, x_out=B, q=B + 1200, x_stride=400, delta_stride=800, x_out_stride=400, q_stride=1600), NO_DEVICE),
    (dict(x=B, delta=B + 400, x_out=B + 800, q=B + 992, x_stride=400, delta_stride=800, x_out_stride=400, q_stride=1600), REFUSED),   # x_out's last values
    (dict(x=B, delta=B + 800, x_out=B + 992, x_stride=400, delta_stride=800, x_out_stride=400), REFUSED),                            # delta's
    (dict(x=B, x_out=B + 400, x_stride=400, x_out_stride=500), REFUSED),                      # distances that differ: by their extent
    (dict(x=B, q=B + 400, x_stride=400, q_stride=3200), REFUSED),
])
def test_rows(built_lib, pkg, changes, code):
    assert _call(built_lib, "attn_rmsnorm_i8", _rows_args(pkg.binding), **changes) == code


@pytest.mark.parametrize("changes,code", [
    (dict(a=B, out=B + 80, a_stride=480, ldc=120), NO_DEVICE),
    (dict(a=B, out=B + 68, a_stride=480, ldc=120), REFUSED),          # a's last two bytes
    (dict(a=B, out=B + 84, a_stride=480, ldc=120), REFUSED),          # the next row's first four
    (dict(w=B, out=B + 80, w_stride=480, ldc=120), NO_DEVICE),
    (dict(a=B, out=B + 80, a_stride=480, ldc=240), REFUSED),          # distances that differ: by their extent
])
def test_products(built_lib, pkg, changes, code):
    assert _call(built_lib, "attn_gemm_i8", _gemm_args(pkg.binding), **changes) == code
