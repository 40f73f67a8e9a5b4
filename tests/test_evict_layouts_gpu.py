"""Eviction over caches that interleave in one buffer: the same as over dense ones of their own."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(built_lib, pkg):
    from llm_infer_b200 import context
    return context


@pytest.mark.parametrize("B,T,keep,Hkv,D", [(1, 60, 17, 2, 64), (3, 60, 17, 2, 64), (5, 3000, 1500, 4, 128)])
def test_interleaved_caches(ctx, B, T, keep, Hkv, D):
    g = torch.Generator(device="cuda").manual_seed(T)
    k, v = (torch.randn((B, T, Hkv, D), generator=g, device="cuda").half() for _ in range(2))
    scores = torch.rand((B, Hkv, T), generator=g, device="cuda")
    lens = torch.randint(1, T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    lens[0] = T
    want = [torch.full((B, T, Hkv, D), 3.0, dtype=torch.float16, device="cuda") for _ in range(2)] + [torch.zeros((B, Hkv, T), device="cuda")]
    want_kept, want_len = ctx.kv_evict(k, v, scores, lens, keep, sink=3, recent=5, out=tuple(want))

    def layouts():
        # sequences outermost, then layers, rows, K and V: input and output are two layers
        stack = torch.full((B, 2, T, 2, Hkv, D), 3.0, dtype=torch.float16, device="cuda")
        yield stack[:, 0, :, 0], stack[:, 0, :, 1], stack[:, 1, :, 0], stack[:, 1, :, 1]
        # rows outermost, then sequences: input, output, K and V side by side
        stack = torch.full((T, B, 4, Hkv, D), 3.0, dtype=torch.float16, device="cuda").transpose(0, 1)
        yield stack[:, :, 0], stack[:, :, 1], stack[:, :, 2], stack[:, :, 3]

    for ki, vi, ko, vo in layouts():
        ki.copy_(k), vi.copy_(v)
        both = torch.zeros((B, Hkv, 2, T), device="cuda")
        both[:, :, 0] = scores
        kept, length = ctx.kv_evict(ki, vi, both[:, :, 0], lens, keep, sink=3, recent=5, out=(ko, vo, both[:, :, 1]))
        for x, y in zip((ko, vo, both[:, :, 1], kept, length, ki, vi, both[:, :, 0]), (*want, want_kept, want_len, k, v, scores)):
            assert torch.equal(x, y)
        ctx.kv_evict(ki, vi, both[:, :, 0], lens, keep, sink=3, recent=5)  # in place
        for b in range(B):
            n = min(int(lens[b]), keep)
            assert torch.equal(ki[b, :n], want[0][b, :n]) and torch.equal(vi[b, :n], want[1][b, :n])
        assert torch.equal(both[:, :, 0], want[2]) and torch.equal(ko, want[0])
