"""What is not a number in the shared decode's operands: it shows in the outputs that it belongs to, and in no other."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(built_lib, pkg):
    from llm_infer_b200 import context
    return context


NAN_SHAPES = [
    # B, H, Hkv, D, P, T: the merge by slices of a row, by a warp a row, by whole rows of many pieces; the prefix kernel
    (2, 8, 2, 64, 100, 30),
    (40, 32, 8, 128, 0, 50),
    (16, 32, 8, 128, 4096, 64),
    (64, 32, 8, 128, 8000, 20),
]


@pytest.mark.parametrize("shape", NAN_SHAPES, ids=lambda s: "b%d_h%d_%d_d%d_p%d_t%d" % s)
@pytest.mark.parametrize("dtype,out_type", [(torch.float16, torch.float16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("scored", [False, True])
def test_what_is_not_a_number_stays_so_and_stays_where_it_is(ctx, shape, dtype, out_type, scored):
    """A query of NaN (all of its scores are NaN) and a valid key of NaN or of +inf scores: the rows that meet them are NaN, their log-sum-exps and
    weights too; every other row is what it is without them."""
    B, H, Hkv, D, P, T = shape
    G = H // Hkv
    g = torch.Generator(device="cuda").manual_seed(B)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)  # noqa: E731
    q, k, v = rand(B, H, D), rand(B, T, Hkv, D), rand(B, T, Hkv, D)
    kp, vp = (rand(P, Hkv, D), rand(P, Hkv, D)) if P else (None, None)
    q[0, :] = q[0, :].abs()
    lens = torch.full((B,), T, dtype=torch.int32, device="cuda")

    def run():
        lse = torch.zeros((B, H), device="cuda")
        scores = torch.zeros((B, Hkv, T), device="cuda") if scored else None
        out = ctx.attn_decode_shared(q, kp, vp, k, v, lens, lse=lse, out_dtype=out_type, scores=scores)
        return out, lse, scores

    clean = run()
    bad = torch.zeros((B, H), dtype=torch.bool, device="cuda")
    q[1, 3] = math.nan
    bad[1, 3] = True
    k[0, T - 1, Hkv - 1, 7] = math.inf  # the queries of sequence 0 are positive: scores of +inf
    bad[0, (Hkv - 1) * G:] = True
    k[B - 1, 2, 0, 5] = math.nan
    bad[B - 1, :G] = True
    if P:
        kp[P // 2, 1, 9] = math.nan
        bad[:, G:2 * G] = True
    out, lse, scores = run()
    assert torch.equal(out.isnan().all(-1), bad) and torch.equal(out.isnan().any(-1), bad)
    assert torch.equal(lse.isnan(), bad)
    assert torch.equal(out[~bad], clean[0][~bad]) and torch.equal(lse[~bad], clean[1][~bad])
    if scored:
        bad_kv = bad.view(B, Hkv, G).any(-1)
        assert bool(scores[bad_kv].isnan().all()) and torch.equal(scores[~bad_kv], clean[2][~bad_kv])
