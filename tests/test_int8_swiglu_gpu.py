"""SwiGLU behind the 8-bit product over every gate that fp32 holds, in each form of the kernel."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"

GATES = [0.0, -0.0, 1e-38, -1e-38, 1e-9, -1e-9, 0.5, -0.5, -17.0, 17.0, -80.0, -87.0, -87.3, -87.34, -87.9, -88.0, -88.5, -88.72, -88.73, -89.0,
         -95.0, -103.0, -104.5, -200.0, -1e9, -3e38, 88.0, 100.0, 1e9]
UPS = [1.0, -1.0, 1e30, -3e-5]


@pytest.mark.parametrize("m,k", [(1, 1), (1, 4096), (20, 8192), (40, 100), (64, 16384), (130, 64), (700, 300)])
def test_gates_of_any_size(built_lib, pkg, m, k):
    """One product of 1 in each sum, so that gate and up are the channels' scales. Against the definition in 64 bits. Rounded are: exp, good to
    two units in the last place (2^-22; below the normal numbers two steps of 2^-149), times the gate (2^-24, or 2^-150), 1 + exp (2^-24),
    the quotient, good to two units (2^-22, or 2^-148), and the product with up (2^-24, or 2^-150)."""
    from llm_infer_b200 import int8 as i8
    gate = torch.tensor(GATES, device=DEV).repeat_interleave(len(UPS))
    up = torch.tensor(UPS, device=DEV).repeat(len(GATES))
    keep = (gate.double() * up.double()).abs() < 3e38  # (products past fp32's range)
    gate, up = gate[keep], up[keep]
    n = gate.numel()
    a, w = i8.rows_i8(m, k), i8.rows_i8(2 * n, k)
    a.zero_(), w.zero_()
    a[:, k // 2] = 1
    w[:, k // 2] = 1
    one = torch.ones(m, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = i8.gemm_i8(a, one, w, torch.cat([gate, up]), swiglu=True, status=status)
    torch.cuda.synchronize()
    assert int(status.item()) == 0
    g, u = gate.double(), up.double()
    want = g / (1.0 + torch.exp(-g)) * u
    bound = want.abs() * (2 * 2.0 ** -22 + 3 * 2.0 ** -24) * 1.01 + (g.abs().clamp_max(200.0) + 2) * 2.0 ** -148 * u.abs() + 2.0 ** -149
    far = (out.double() - want).abs() - bound
    assert (far <= 0).all(), [(float(gate[j]), float(up[j]), float(out[0, j]), float(want[j])) for j in (far[0] > 0).nonzero()[:, 0].tolist()]


@pytest.mark.parametrize("m", [1, 300])
def test_gates_that_are_no_numbers(built_lib, pkg, m):
    """The gate's infinity is the product's, and NaN stays in its channel."""
    from llm_infer_b200 import int8 as i8
    gate = torch.tensor([float("inf"), float("nan"), 1.0, -88.0], device=DEV)
    a, w = i8.rows_i8(m, 16), i8.rows_i8(8, 16)
    a.zero_(), w.zero_()
    a[:, 0] = 1
    w[:, 0] = 1
    out = i8.gemm_i8(a, torch.ones(m, device=DEV), w, torch.cat([gate, torch.ones(4, device=DEV)]), swiglu=True)
    torch.cuda.synchronize()
    assert torch.isposinf(out[:, 0]).all() and torch.isnan(out[:, 1]).all() and torch.isfinite(out[:, 2:]).all()
