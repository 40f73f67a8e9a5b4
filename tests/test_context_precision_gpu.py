"""Probabilities of the shared decode to the last bits that its parts of 16 bits hold.

An fp16 probability is lifted by 2^7 (it is at most 2^8 relative to the running maximum, fp16 ends at 2^16), so that fp16's smallest
spacing, 2^-24, is 2^-31 of a probability relative to a piece's maximum; rounding to it is off by 2^-32 at most. bf16 has fp32's range."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
GRID = {torch.float16: 2.0 ** -32, torch.bfloat16: 0.0}


@pytest.fixture(scope="module")
def ctx(built_lib, pkg):
    from llm_infer_b200 import context
    return context


def _two_keys(dtype, B, H, Hkv, D, n, top, small, most):
    """Caches [n, Hkv, D] whose key `top` has score 0 and value 0 and whose key `small[head]` has score -a and value 1; all others have
    score -64 and value 0. a differs from query row to query row, up to `most`."""
    a = ((1 + torch.arange(B * H, dtype=torch.float64)) * (most / (B * H))).to(dtype).cuda()  # steps exact in either type
    q = torch.zeros((B, H, D), dtype=dtype, device="cuda")
    q[:, :, 0], q[:, :, 1] = a.view(B, H), 8
    k, v = torch.zeros((n, Hkv, D), dtype=dtype, device="cuda"), torch.zeros((n, Hkv, D), dtype=dtype, device="cuda")
    k[:, :, 1] = -8
    k[top, :, 1] = 0
    for h, at in enumerate(small):
        k[at, h, 0], k[at, h, 1], v[at, h] = -1, 0, 1
    return q, k, v, a.double().view(B, H, 1)


def _attend(ctx, form, q, k, v, **kw):
    B, Hkv, D = q.shape[0], k.shape[1], k.shape[2]
    if form == "own":
        return ctx.attn_decode_shared(q, None, None, k[None].expand(B, -1, -1, -1).contiguous(), v[None].expand(B, -1, -1, -1).contiguous(), **kw)
    none = torch.zeros((B, 0, Hkv, D), dtype=q.dtype, device="cuda")
    return ctx.attn_decode_shared(q, k, v, none, none, **kw)


# own rows; a prefix in the split pass; a prefix long enough for the tensor cores' kernel (128 query rows per kv head)
FORMS = {"own": (4, 64, 2, 70), "prefix": (4, 64, 2, 300), "long prefix": (16, 128, 16, 16384)}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("D", [64, 128])
def test_fp32_outputs_take_probabilities_in_full_at_every_key_of_a_block(ctx, dtype, form, D):
    """a up to 2: p / (1 + p) within 6.25 * 2^-22: exp2 2^-22 and the scale's product 2^-22 of p, the sum 2^-24, the division 2^-23, three
    cut-off additions 2^-23 each, the joining of pieces 2^-21; and 2^-22 for the exponent that the lift rounds at 7 (half of 2^-21 times
    ln 2, for both probabilities: 1.4 * 2^-22), together 7.75 * 2^-22. The small key's place in its block of 64 goes by the kv head."""
    B, H, Hkv, n = FORMS[form]
    for first in range(0, 64, Hkv * 4):
        small = [(n // 2 // 64) * 64 - 64 + (first + 4 * h + h % 4) % 64 for h in range(Hkv)] if n > 128 else [(first + 4 * h) % 64 for h in range(Hkv)]
        q, k, v, a = _two_keys(dtype, B, H, Hkv, D, n, n - 1, small, 2.0)
        out = _attend(ctx, form, q, k, v, out_dtype=torch.float32, scale=0.75).double()
        p = torch.exp(-0.75 * a)
        want = (p / (1 + p)).expand(B, H, D)
        assert float(((out - want) / want).abs().max()) <= 7.75 * 2.0 ** -22


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("form", list(FORMS))
def test_fp32_outputs_keep_small_probabilities(ctx, dtype, form):
    """a up to 16, the only value on the small key: p / (1 + p) to the roundings of an exponent of up to 30 (scale in log2 units 2^-24 of
    it, its own half spacing 2^-20; times ln 2: 2.0 * 2^-20), exp2 2^-22 and the few of the sum and the joining (5 * 2^-22), and what the
    grid of the parts leaves of p."""
    B, H, Hkv, n = FORMS[form]
    for first in (6, 40):  # own rows: in the piece of the large key, and in another one
        q, k, v, a = _two_keys(dtype, B, H, Hkv, 128, n, 3, [first + h for h in range(Hkv)], 16.0)
        out = _attend(ctx, form, q, k, v, out_dtype=torch.float32, scale=1.0).double()
        p = torch.exp(-a)
        want = (p / (1 + p)).expand(B, H, 128)
        assert bool(((out - want).abs() <= (4 * 2.0 ** -20 + GRID[dtype] / p) * want).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("form", list(FORMS))
def test_16_bit_outputs_keep_many_small_probabilities(ctx, dtype, form):
    """One key takes most of the weight and has value 0, all others have probability e^-17 of its and value 1: together
    (n - 1) e^-17, which the sum has and the product must not lose. P is rounded once: u of the type, or half of its smallest spacing."""
    B, H, Hkv, n = FORMS[form]
    D = 128
    q = torch.zeros((B, H, D), dtype=dtype, device="cuda")
    q[:, :, 0] = 17
    k, v = torch.zeros((n, Hkv, D), dtype=dtype, device="cuda"), torch.ones((n, Hkv, D), dtype=dtype, device="cuda")
    k[:, :, 0] = -1
    k[5, :, 0], v[5] = 0, 0
    u, p = torch.finfo(dtype).eps / 2, math.exp(-17.0)
    small = 2.0 ** -25 if dtype == torch.float16 else 0.0  # of fp16 outputs below 2^-14
    want = (n - 1) * p / (1 + (n - 1) * p)
    out = _attend(ctx, form, q, k, v, scale=1.0).double()
    assert float((out - want).abs().max()) <= (2 * u + GRID[dtype] / p + 4 * 2.0 ** -20) * want + small
