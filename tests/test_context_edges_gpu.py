"""Long-context operators at the edges of their contracts: operands that the launch in front has just written."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(built_lib, pkg):
    from llm_infer_b200 import context
    return context


@pytest.mark.parametrize("dtype,out_type", [(torch.float16, torch.float16), (torch.bfloat16, torch.float32)])
def test_long_prefix_decode_right_behind_the_kernels_that_write_its_operands(ctx, dtype, out_type):
    """Queries, cache rows and lengths come from launches directly in front of the call (rotary positions and insert, eviction in
    place), none of which it waits for on the host: in a graph and in a row the results are those of calls with a wait between all."""
    B, H, Hkv, D, P, T, steps = 40, 32, 8, 128, 5000, 60, 6
    g = torch.Generator(device="cuda").manual_seed(21)
    rand = lambda *s, dtype=dtype: torch.randn(s, generator=g, device="cuda").to(dtype)  # noqa: E731
    stacks = [rand(B, H + 2 * Hkv, D, dtype=torch.float32) for _ in range(steps)]
    kp, vp, k0, v0 = rand(P, Hkv, D), rand(P, Hkv, D), rand(B, T, Hkv, D), rand(B, T, Hkv, D)
    inv_freq = ctx.rope_frequencies(D, 10000.0)[0].cuda()
    lens0 = torch.randint(20, T, (B,), generator=g, device="cuda", dtype=torch.int32)
    pos = P + torch.arange(B, dtype=torch.int32, device="cuda")
    k, v, lens = k0.clone(), v0.clone(), lens0.clone()
    scores = torch.zeros((B, Hkv, T), device="cuda")
    row = torch.zeros_like(lens)
    ws = ctx.SharedWorkspace(B, H, Hkv, D, rows=T)
    outs = [torch.zeros((B, H, D), dtype=out_type, device="cuda") for _ in range(2 * steps)]

    def run(wait):
        k.copy_(k0), v.copy_(v0), lens.copy_(lens0), scores.zero_()
        for i, s in enumerate(stacks):
            row.copy_(lens)
            lens.add_(1)
            wait()
            q = ctx.rope_positions(s[:, :H], s[:, H:H + Hkv], s[:, H + Hkv:], k, v, pos, row, inv_freq=inv_freq, q_out_dtype=dtype)
            wait()
            ctx.attn_decode_shared(q, kp, vp, k, v, lens, out=outs[2 * i], scores=scores, workspace=ws)
            wait()
            ctx.kv_evict(k, v, scores, lens, 18 - i, sink=2, recent=5, kv_len_out=lens)
            wait()
            ctx.attn_decode_shared(q, kp, vp, k, v, lens, out=outs[2 * i + 1], scores=scores, workspace=ws)
            wait()
        torch.cuda.synchronize()
        return [x.clone() for x in (*outs, k, v, scores, lens)]

    want = run(torch.cuda.synchronize)
    launches = ctx._b.load().attn_kernel_launch_count()
    got = run(lambda: None)
    assert ctx._b.load().attn_kernel_launch_count() - launches == steps * (1 + 2 + 2 + 2)  # (the long prefix's kernel, and the merge)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        k.copy_(k0), v.copy_(v0), lens.copy_(lens0), scores.zero_()
        for i, s in enumerate(stacks):
            row.copy_(lens)
            lens.add_(1)
            q = ctx.rope_positions(s[:, :H], s[:, H:H + Hkv], s[:, H + Hkv:], k, v, pos, row, inv_freq=inv_freq, q_out_dtype=dtype)
            ctx.attn_decode_shared(q, kp, vp, k, v, lens, out=outs[2 * i], scores=scores, workspace=ws)
            ctx.kv_evict(k, v, scores, lens, 18 - i, sink=2, recent=5, kv_len_out=lens)
            ctx.attn_decode_shared(q, kp, vp, k, v, lens, out=outs[2 * i + 1], scores=scores, workspace=ws)
    for _ in range(3):
        for x in (*outs, k, v, lens):
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((*outs, k, v, scores, lens), want))
    assert int(ws.status.item()) == 0
