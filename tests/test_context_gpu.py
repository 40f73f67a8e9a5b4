"""Rotary positions, shared-prefix decode with accumulated weights, and eviction against their definitions in 64 bits.

Tolerances follow from the number formats, element by element. u is half a unit in the last place of a type (fp16 2^-11,
bf16 2^-8, fp32 2^-24): finfo.eps / 2.
* rope: two products and a sum of fp32, cos and sin within 2^-22, then one rounding: u_out |y| + 2^-21 factor (|a| + |b|).
* decode: scores are sums of head_dim exact products in fp32, off by ds = (D / 16 + 8) 2^-23 scale sum|q k| at most; a probability
  is then off by a factor of 2 ds + 2^-20 (exponential, sums of the softmax), and by u_P where it is rounded to the caches' type
  (16-bit outputs) or 2 u_P^2 where its residual is carried along (fp32 outputs). A = sum p |v| bounds what that does:
  u_out |o| + (u_P + 2 ds + 2^-20) A. Weights: (2 ds + 2^-20) w + 2^-23 |score|.
* eviction copies: equal."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = {name: torch.finfo(t).eps / 2 for name, t in T.items()}


@pytest.fixture(scope="module")
def ctx(built_lib, pkg):
    from llm_infer_b200 import context
    return context


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------------------------------------------------- rotary
def _rope64(x, pos, inv_freq, factor, layout):
    x, R = x.double(), 2 * inv_freq.numel()
    a = pos.double()[:, None] * inv_freq.double()[None, :]
    c, s = (torch.cos(a) * factor)[:, None], (torch.sin(a) * factor)[:, None]
    y, mag = x.clone(), x.abs()
    i0, i1 = (slice(0, R // 2), slice(R // 2, R)) if layout == "half" else (slice(0, R, 2), slice(1, R, 2))
    y[..., i0], y[..., i1] = x[..., i0] * c - x[..., i1] * s, x[..., i0] * s + x[..., i1] * c
    mag[..., i0] = mag[..., i1] = (x[..., i0].abs() + x[..., i1].abs()) * factor
    return y, mag


@pytest.mark.parametrize("N,H,Hkv,D,R,layout,types,first", [
    (1, 32, 8, 128, 128, "half", ("f32", "f16", "f16"), 0),
    (8, 32, 4, 64, 64, "interleaved", ("f32", "f32", "f16"), 131071),
    (7, 8, 2, 128, 64, "half", ("bf16", "bf16", "bf16"), 100003),
    (131, 24, 2, 128, 32, "interleaved", ("f16", "f16", "f16"), 5000),
    (5000, 4, 4, 64, 64, "half", ("bf16", "f32", "bf16"), 0),
    (33, 3, 1, 80, 24, "half", ("f16", "bf16", "f16"), 17),          # 24 is no multiple of 16: single values
    (33, 5, 5, 96, 32, "interleaved", ("f32", "f16", "bf16"), 17),
    (3, 2, 1, 6, 2, "interleaved", ("f16", "f32", "f16"), 2 ** 30),
])
def test_rope_positions(ctx, N, H, Hkv, D, R, layout, types, first):
    tin, tq, tc = types
    g = _gen(N + D)
    stack = torch.randn((N, H + 2 * Hkv, D), generator=g).to(T[tin])
    inv_freq, factor = ctx.rope_frequencies(R, 500000.0, {"type": "yarn", "factor": 4.0, "original": 8192})
    pos = first + torch.arange(N, dtype=torch.int32) * 3
    B = min(N, 3)
    seq = torch.arange(N, dtype=torch.int32) % B
    row = torch.arange(N, dtype=torch.int32) // B + 1
    rows = int(row.max()) + 2
    kc = torch.full((B, rows, Hkv, D), 7.0, dtype=T[tc], device="cuda")
    vc = kc.clone()
    dev = stack.cuda()
    q, k, v = dev[:, :H], dev[:, H:H + Hkv], dev[:, H + Hkv:]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = ctx.rope_positions(q, k, v, kc, vc, pos.cuda(), row.cuda(), seq=seq.cuda(), inv_freq=inv_freq.cuda(), factor=factor,
                             layout=layout, q_out_dtype=T[tq], status=status)
    torch.cuda.synchronize()
    want, mag = _rope64(stack[:, :H], pos, inv_freq, factor, layout)
    assert out.dtype == T[tq]
    err = (out.double().cpu() - want).abs()
    assert (err <= U[tq] * want.abs() + 2.0 ** -21 * mag).all(), err.max()
    want, mag = _rope64(stack[:, H:H + Hkv], pos, inv_freq, factor, layout)
    got = kc.cpu().double()[seq.long(), row.long()]
    assert ((got - want).abs() <= U[tc] * want.abs() + 2.0 ** -21 * mag).all()
    assert torch.equal(vc.cpu()[seq.long(), row.long()], stack[:, H + Hkv:].float().to(T[tc]))
    untouched = torch.ones((B, rows), dtype=torch.bool)
    untouched[seq.long(), row.long()] = False
    assert (kc.cpu()[untouched] == 7).all() and (vc.cpu()[untouched] == 7).all()
    assert int(status.item()) == 0


def test_rope_positions_in_place_unaligned_and_rows_that_do_not_exist(ctx):
    g = _gen(3)
    N, H, Hkv, D = 6, 4, 2, 64
    flat = torch.randn(N * (H + 2 * Hkv) * D + 1, generator=g).half().cuda()
    stack = flat[1:].view(N, H + 2 * Hkv, D)  # two bytes off every vector boundary
    before = stack.cpu().clone()
    kc, vc = (torch.zeros((2, 4, Hkv, D), dtype=torch.float16, device="cuda") for _ in range(2))
    inv_freq, _ = ctx.rope_frequencies(D, 10000.0)
    pos = torch.tensor([0, 1, 2, 3, 4, 5], dtype=torch.int32)
    row = torch.tensor([0, 1, 3, 4, -1, 2], dtype=torch.int32)  # 4 and -1 do not exist
    seq = torch.tensor([0, 1, 0, 1, 0, 2], dtype=torch.int32)   # nor does sequence 2
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    q = stack[:, :H]
    out = ctx.rope_positions(q, stack[:, H:H + Hkv], stack[:, H + Hkv:], kc, vc, pos.cuda(), row.cuda(), seq=seq.cuda(),
                             inv_freq=inv_freq.cuda(), layout="half", q_out=q, status=status)
    assert out.data_ptr() == q.data_ptr()
    want, mag = _rope64(before[:, :H], pos, inv_freq, 1.0, "half")
    assert ((q.double().cpu() - want).abs() <= U["f16"] * want.abs() + 2.0 ** -21 * mag).all()
    assert torch.equal(stack[:, H:].cpu(), before[:, H:])
    assert int(status.item()) == 2
    there = torch.zeros((2, 4), dtype=torch.bool)
    there[0, 0] = there[1, 1] = there[0, 3] = True
    assert (vc.cpu()[~there] == 0).all() and (kc.cpu()[~there] == 0).all()
    assert torch.equal(vc.cpu()[seq[:3].long(), row[:3].long()], before[:3, H + Hkv:])


def test_rope_positions_of_default_frequencies_match_the_engines_insert(ctx):
    """Interleaved, unscaled, short positions: what rope_kv_insert writes, within the fp32 rounding of its angle."""
    from llm_infer_b200 import attention
    g = _gen(9)
    B, H, Hkv, D = 3, 8, 2, 128
    q, k, v = (torch.randn((B, n, D), generator=g).cuda() for n in (H, Hkv, Hkv))
    pos, row = torch.tensor([0, 5, 900], dtype=torch.int32).cuda(), torch.tensor([0, 5, 9], dtype=torch.int32).cuda()
    caches = [torch.zeros((B, 10, Hkv, D), dtype=torch.float16, device="cuda") for _ in range(4)]
    want = attention.rope_kv_insert(q, k, v, caches[0], caches[1], pos, row, theta=10000.0)
    inv_freq, _ = ctx.rope_frequencies(D, 10000.0)
    got = ctx.rope_positions(q, k, v, caches[2], caches[3], pos, row, inv_freq=inv_freq.cuda())
    # the angle's rounding: 900 * 2^-24, times the pair's length (at most 6 here)
    assert (got - want).abs().max() <= 6 * 1000 * 2.0 ** -24
    assert torch.equal(caches[1], caches[3])
    assert (caches[0].float() - caches[2].float()).abs().max() <= 2.0 ** -9  # one fp16 step below 4


# ------------------------------------------------------------------------------------------------- shared-prefix decode
def _decode64(q, kp, vp, k, v, lens, scale):
    """out, bound A, ds, weights [B, Hkv, T], lse in 64 bits."""
    B, H, D = q.shape
    Hkv, Tn = k.shape[2], k.shape[1]
    G = H // Hkv
    out, A = torch.zeros((B, H, D), dtype=torch.float64), torch.zeros((B, H, D), dtype=torch.float64)
    ds, lse = torch.zeros((B, H, 1), dtype=torch.float64), torch.full((B, H), -math.inf, dtype=torch.float64)
    w = torch.zeros((B, Hkv, Tn), dtype=torch.float64)
    P = 0 if kp is None else kp.shape[0]
    for b in range(B):
        n = int(lens[b])
        if P + n == 0:
            continue
        for h in range(Hkv):
            kk, vv = k[b, :n, h].double(), v[b, :n, h].double()
            if P:
                kk, vv = torch.cat([kp[:, h].double(), kk]), torch.cat([vp[:, h].double(), vv])
            qq = q[b, h * G:(h + 1) * G].double()
            s = qq @ kk.T * scale
            p = torch.softmax(s, 1)
            sl = slice(h * G, (h + 1) * G)
            out[b, sl], A[b, sl] = p @ vv, p @ vv.abs()
            ds[b, sl, 0] = ((qq.abs() @ kk.abs().T) * abs(scale)).amax(1) * (D / 16 + 8) * 2.0 ** -23
            lse[b, sl] = torch.logsumexp(s, 1)
            w[b, h, :n] = p[:, P:].sum(0)
    return out, A, ds, w, lse


def _check_decode(ctx, B, H, Hkv, D, P, Tn, lens, dtype, out_type, scored, seed=1, scale=0.0, std=1.5, **kw):
    g = _gen(seed)
    mk = lambda *s, std=1.0: (torch.randn(s, generator=g) * std).to(T[dtype])  # noqa: E731
    q, k, v = mk(B, H, D, std=std), mk(B, Tn, Hkv, D), mk(B, Tn, Hkv, D)
    kp, vp = (mk(P, Hkv, D), mk(P, Hkv, D)) if P else (None, None)
    want, A, ds, w, want_lse = _decode64(q, kp, vp, k, v, lens, scale or D ** -0.5)
    for b, n in enumerate(lens):  # what lies behind a length must not matter
        k[b, n:], v[b, n:] = float("nan"), float("inf")
    before = torch.rand((B, Hkv, Tn), generator=g)
    c = lambda t: None if t is None else t.cuda()  # noqa: E731
    lse = torch.full((B, H), 99.0, device="cuda")
    scores = c(before) if scored else None
    scores_out = torch.full((B, Hkv, Tn), -5.0, device="cuda") if scored else None
    ws = ctx.SharedWorkspace(B, H, Hkv, D, rows=Tn if scored else 0)
    for _ in range(2):  # the workspace is reused as it is
        out = ctx.attn_decode_shared(c(q), c(kp), c(vp), c(k), c(v), torch.tensor(lens, dtype=torch.int32, device="cuda"), lse=lse,
                                     out_dtype=T[out_type], scale=scale, scores=scores, scores_out=scores_out, workspace=ws, **kw)
    torch.cuda.synchronize()
    assert int(ws.status.item()) == 0
    got = out.double().cpu()
    u_p = U[dtype] if out_type != "f32" else 2 * U[dtype] ** 2
    ok = (got - want).abs() <= U[out_type] * want.abs() + (u_p + 2 * ds + 2.0 ** -20) * A
    assert ok.all(), (got - want).abs().max()
    got_lse = lse.double().cpu()
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(got_lse), empty) and (got_lse[empty] < 0).all()
    assert ((got_lse - want_lse).abs()[~empty] <= (ds[..., 0] + 2.0 ** -18 * (1 + want_lse.abs()))[~empty]).all()
    if scored:
        gs = scores_out.double().cpu()
        valid = torch.arange(Tn)[None, None, :] < torch.tensor(lens)[:, None, None]
        valid = valid.expand(B, Hkv, Tn)
        limit = (2 * ds.view(B, Hkv, -1).amax(2)[..., None] + 2.0 ** -20) * w + 2.0 ** -23 * (before.double() + w)
        assert ((gs - before.double() - w).abs() <= limit)[valid].all()
        assert (gs[~valid] == -5.0).all()


SHAPES = [
    # B, H, Hkv, D, P, T, lens
    (1, 32, 8, 128, 0, 1, [1]),
    (1, 32, 8, 128, 1, 1, [0]),
    (2, 32, 8, 128, 0, 70, [0, 70]),                     # an empty row beside a full one
    (3, 8, 2, 128, 17, 33, [33, 0, 1]),
    (2, 32, 4, 64, 512, 64, [64, 13]),
    (1, 16, 16, 64, 100, 65, [65]),
    (5, 24, 2, 128, 130, 200, [200, 16, 17, 15, 1]),     # twelve heads per kv head
    (16, 32, 8, 128, 1000, 97, [(i * 37) % 98 for i in range(16)]),
    (17, 8, 8, 64, 333, 50, [(i * 13) % 51 for i in range(17)]),   # 17 prefix rows per kv head: two blocks
    (40, 8, 1, 128, 301, 40, [(i * 7) % 41 for i in range(40)]),   # 320 prefix rows on one kv head
    (3, 32, 1, 64, 129, 77, [77, 76, 3]),                # 32 heads per kv head
    (2, 40, 1, 128, 65, 66, [66, 2]),                    # 40
    (2, 64, 1, 128, 0, 129, [129, 128]),                 # 64
    (4, 9, 3, 128, 70, 40, [40, 39, 0, 5]),              # three kv heads: no groups of two or four
    (130, 4, 2, 64, 5, 9, [(i * 5) % 10 for i in range(130)]),
    (1, 32, 8, 128, 20000, 3000, [2999]),
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "b%d_h%d_%d_d%d_p%d_t%d" % s[:6])
@pytest.mark.parametrize("dtype,out_type", [("f16", "f16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f32")])
@pytest.mark.parametrize("scored", [False, True])
def test_decode_shared(ctx, shape, dtype, out_type, scored):
    _check_decode(ctx, *shape, dtype, out_type, scored)


# long prefixes and many query rows: the prefix as a matrix product on the tensor cores
TENSOR_SHAPES = [
    # B, H, Hkv, D, P, T, lens
    (5, 32, 8, 128, 513, 20, [20, 3, 0, 7, 1]),
    (32, 32, 8, 128, 1024, 10, [(i * 3) % 11 for i in range(32)]),       # 128 rows: exactly a tile
    (43, 24, 8, 64, 2049, 10, [(i * 3) % 11 for i in range(43)]),        # 129 rows, one key in the last block
    (130, 4, 2, 64, 4095, 9, [(i * 5) % 10 for i in range(130)]),        # 260 rows: two segments per kv head
    (100, 12, 4, 128, 1999, 5, [(i * 5) % 6 for i in range(100)]),       # 300 rows: the last segment has one tile
    (3, 24, 2, 128, 5000, 70, [70, 1, 0]),
    (7, 40, 5, 64, 1000, 33, [33] * 7),
    (65, 8, 1, 128, 20000, 3, [3, 0, 1] * 21 + [2, 2]),
    (2, 64, 1, 128, 65, 129, [129, 128]),
    (300, 8, 1, 64, 10000, 4, [i % 5 for i in range(300)]),              # 2400 rows: ten segments
]


@pytest.mark.parametrize("shape", TENSOR_SHAPES, ids=lambda s: "b%d_h%d_%d_d%d_p%d_t%d" % s[:6])
@pytest.mark.parametrize("dtype,out_type,scored", [("f16", "f16", True), ("bf16", "bf16", False), ("f16", "f32", False), ("bf16", "f32", True)])
def test_decode_shared_long_prefix(ctx, shape, dtype, out_type, scored):
    _check_decode(ctx, *shape, dtype, out_type, scored)


def test_decode_shared_long_prefix_large_scores(ctx):
    _check_decode(ctx, 9, 32, 8, 128, 3000, 100, [100, 50, 1, 0, 5, 6, 7, 8, 9], "f16", "f16", True, std=20.0)
    _check_decode(ctx, 9, 32, 8, 128, 3000, 100, [100, 50, 1, 0, 5, 6, 7, 8, 9], "bf16", "f32", True, scale=0.5)
    _check_decode(ctx, 9, 32, 8, 128, 3000, 100, [100, 50, 1, 0, 5, 6, 7, 8, 9], "f16", "f32", True, scale=-0.1)


def test_decode_shared_large_scores_and_a_given_scale(ctx):
    """One key takes everything: the running maximum moves by hundreds, probabilities underflow."""
    _check_decode(ctx, 4, 8, 2, 128, 500, 100, [100, 50, 1, 0], "f16", "f16", True, std=20.0)
    _check_decode(ctx, 4, 8, 2, 128, 500, 100, [100, 50, 1, 0], "f16", "f32", True, scale=0.5)


def test_decode_shared_nothing_to_attend(ctx):
    q = torch.randn(2, 4, 64, device="cuda").half()
    for rows, lens in ((0, None), (3, 0)):
        kv = torch.full((2, rows, 2, 64), float("nan"), device="cuda").half()
        lse = torch.zeros((2, 4), device="cuda")
        out = ctx.attn_decode_shared(q, None, None, kv, kv.clone(), lens, lse=lse)
        assert (out == 0).all() and (lse == -math.inf).all()


def test_decode_shared_strided_operands_and_long_offsets(ctx):
    """Rows and sequences at other distances, and caches whose offsets pass 32 bits (elements and bytes)."""
    g = torch.Generator(device="cuda").manual_seed(4)
    B, H, Hkv, D, Tn = 2, 8, 2, 64, 64
    gap = 2 ** 32 + 4096  # elements between the two sequences
    big = torch.empty(gap + 2 * Tn * Hkv * D * 2, dtype=torch.float16, device="cuda")
    k = big.as_strided((B, Tn, Hkv, D), (gap, 2 * Hkv * D, D, 1))
    v = big[Hkv * D:].as_strided((B, Tn, Hkv, D), (gap, 2 * Hkv * D, D, 1))  # K and V rows interleaved
    k.copy_(torch.randn(k.shape, generator=g, device="cuda"))
    v.copy_(torch.randn(k.shape, generator=g, device="cuda"))
    pre = torch.randn((50, 2, Hkv, D), generator=g, device="cuda").half()
    kp, vp = pre[:, 0], pre[:, 1]
    q = torch.randn((B, H, D), generator=g, device="cuda").half()
    got = ctx.attn_decode_shared(q, kp, vp, k, v, torch.tensor([64, 31], dtype=torch.int32, device="cuda"))
    want, A, ds, _, _ = _decode64(q.cpu(), kp.cpu(), vp.cpu(), k.cpu(), v.cpu(), [64, 31], D ** -0.5)
    ok = (got.double().cpu() - want).abs() <= U["f16"] * want.abs() + (U["f16"] + 2 * ds + 2.0 ** -20) * A
    assert ok.all()


def test_decode_shared_equals_itself_and_clamps_a_length(ctx):
    g = _gen(6)
    q, k, v = (torch.randn(s, generator=g).half().cuda() for s in ((3, 32, 128), (3, 90, 8, 128), (3, 90, 8, 128)))
    kp, vp = (torch.randn((700, 8, 128), generator=g).half().cuda() for _ in range(2))
    lens = torch.tensor([90, 1000, 7], dtype=torch.int32, device="cuda")
    ws = ctx.SharedWorkspace(3, 32, 8, 128)
    first = ctx.attn_decode_shared(q, kp, vp, k, v, lens, workspace=ws)
    assert int(ws.status.item()) == 2
    for _ in range(5):
        assert torch.equal(ctx.attn_decode_shared(q, kp, vp, k, v, lens, workspace=ws), first)
    lens[1] = 90
    assert torch.equal(ctx.attn_decode_shared(q, kp, vp, k, v, lens), first)


def test_decode_shared_on_another_stream_and_in_a_graph(ctx):
    g = _gen(8)
    q, k, v = (torch.randn(s, generator=g).half().cuda() for s in ((2, 8, 128), (2, 40, 2, 128), (2, 40, 2, 128)))
    scores = torch.zeros((2, 2, 40), device="cuda")
    want = ctx.attn_decode_shared(q, None, None, k, v, 40)
    ws = ctx.SharedWorkspace(2, 8, 2, 128, rows=40)
    out = torch.empty_like(want)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    ctx.attn_decode_shared(q, None, None, k, v, 40, out=out, scores=scores, workspace=ws, stream=side)
    side.synchronize()
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.attn_decode_shared(q, None, None, k, v, 40, out=out, scores=scores, workspace=ws)
    out.zero_()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    assert abs(float(scores.sum().item()) - 4 * 2 * 8) < 1e-3  # four steps, sixteen heads, weights that sum to one


# ------------------------------------------------------------------------------------------------------------ eviction
def _kept64(scores, n, keep, sink, recent):
    """Rows that stay of one head, from the definition: always-kept ones, then by (score descending, row ascending)."""
    if n <= keep:
        return list(range(n))
    s = scores.astype(np.float64)
    order = sorted(range(n), key=lambda i: (not (i < sink or i >= n - recent), bool(np.isnan(s[i])), -s[i] if not np.isnan(s[i]) else 0.0, i))
    return sorted(order[:keep])


def _scores(kind, shape, g):
    s = torch.exp(1.5 * torch.randn(shape, generator=g))
    if kind == "ties":
        s = torch.randint(0, 3, shape, generator=g).float()
    elif kind == "odd":
        s = torch.randn(shape, generator=g)
        pick = torch.randint(0, 12, shape, generator=g)
        for code, val in ((0, math.nan), (1, math.inf), (2, -math.inf), (3, 0.0), (4, -0.0), (5, 1e-42)):
            s[pick == code] = val
    elif kind == "flat":
        s = torch.zeros(shape)
    return s


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("B,Hkv,D,Tn,lens,keep,sink,recent,kind", [
    (1, 8, 128, 1024, [1024], 256, 4, 64, "real"),
    (1, 1, 8, 1, [1], 1, 0, 0, "real"),
    (2, 2, 64, 40, [40, 0], 1, 0, 0, "real"),
    (2, 2, 64, 40, [40, 39], 5, 3, 2, "odd"),               # nothing left to choose
    (3, 4, 64, 700, [700, 300, 299], 300, 4, 50, "ties"),
    (3, 3, 80, 513, [513, 512, 100], 200, 0, 200, "real"),  # only recent rows
    (2, 16, 128, 2500, [2500, 1777], 999, 7, 0, "odd"),
    (2, 2, 128, 5000, [5000, 4097], 4096, 4, 100, "flat"),
    (1, 2, 64, 40000, [39999], 12345, 4, 1000, "ties"),
    (1, 1, 16, 400000, [399991], 30001, 4, 1000, "odd"),    # more keys than a CTA stages
])
def test_kv_evict(ctx, in_place, B, Hkv, D, Tn, lens, keep, sink, recent, kind):
    g = _gen(Tn + keep)
    k, v = (torch.randn((B, Tn, Hkv, D), generator=g).half() for _ in range(2))
    s = _scores(kind, (B, Hkv, Tn), g)
    for b, n in enumerate(lens):
        s[b, :, n:] = math.inf  # stale scores behind the length
    kd, vd, sd = k.cuda(), v.cuda(), s.cuda()
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    T2 = Tn if in_place else keep + 3
    if in_place:
        ko, vo, so, kw = kd, vd, sd, dict(kv_len_out=ln)
    else:
        ko, vo = (torch.full((B, T2, Hkv, D), 9.0, dtype=torch.float16, device="cuda") for _ in range(2))
        so = torch.full((B, Hkv, T2), 9.0, device="cuda")
        kw = dict(out=(ko, vo, so))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    kept, new = ctx.kv_evict(kd, vd, sd, ln, keep, sink=sink, recent=recent, status=status, **kw)
    torch.cuda.synchronize()
    assert int(status.item()) == 0
    assert new.tolist() == [min(n, keep) for n in lens]
    ko, vo, so, kept = ko.cpu(), vo.cpu(), so.cpu(), kept.cpu()
    for b, n in enumerate(lens):
        m = min(n, keep)
        for h in range(Hkv):
            rows = _kept64(s[b, h].numpy(), n, keep, sink, recent)
            assert kept[b, h, :m].tolist() == rows
            assert (kept[b, h, m:] == -1).all()
            assert torch.equal(ko[b, :m, h], k[b, rows, h]) and torch.equal(vo[b, :m, h], v[b, rows, h])
            assert torch.equal(so[b, h, :m].view(torch.int32), s[b, h, rows].view(torch.int32))
        assert (so[b, :, m:] == 0).all()
        if in_place:  # rows behind the old length, and between the lengths, are left alone
            assert torch.equal(ko[b, m:], k[b, m:])
        else:
            assert (ko[b, m:] == 9).all() and (vo[b, m:] == 9).all()
    if not in_place:
        assert torch.equal(kd.cpu(), k) and torch.equal(sd.cpu().view(torch.int32), s.view(torch.int32))


def test_kv_evict_strided_caches_and_a_clamped_length(ctx):
    g = _gen(5)
    kv = torch.randn((2, 100, 2, 4, 64), generator=g).half().cuda()  # K and V rows interleaved
    s = torch.rand((2, 4, 128), generator=g).cuda()[..., :100]
    out = torch.zeros((2, 40, 2, 4, 64), dtype=torch.float16, device="cuda")
    so = torch.zeros((2, 4, 64), device="cuda")[..., :40]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    kept, new = ctx.kv_evict(kv[:, :, 0], kv[:, :, 1], s, torch.tensor([500, 60], dtype=torch.int32, device="cuda"), 33, sink=1,
                             recent=5, out=(out[:, :, 0], out[:, :, 1], so), status=status)
    assert int(status.item()) == 2 and new.tolist() == [33, 33]
    for b, n in enumerate((100, 60)):
        for h in range(4):
            rows = _kept64(s[b, h].cpu().numpy(), n, 33, 1, 5)
            assert kept[b, h].tolist() == rows
            assert torch.equal(out[b, :33, 0, h].cpu(), kv[b, rows, 0, h].cpu()) and torch.equal(out[b, :33, 1, h].cpu(), kv[b, rows, 1, h].cpu())


def test_decode_then_evict_then_decode(ctx):
    """The accumulated weights of a few steps choose the rows; attention over the kept rows is what the definition gives."""
    g = _gen(12)
    B, H, Hkv, D, Tn = 2, 8, 2, 64, 200
    k, v = (torch.randn((B, Tn, Hkv, D), generator=g).half().cuda() for _ in range(2))
    lens = torch.tensor([200, 150], dtype=torch.int32, device="cuda")
    scores = torch.zeros((B, Hkv, Tn), device="cuda")
    for i in range(3):
        ctx.attn_decode_shared(torch.randn((B, H, D), generator=g).half().cuda(), None, None, k, v, lens, scores=scores)
    total = scores.sum((1, 2)).cpu()
    assert (total - 3 * H).abs().max() < 1e-3
    k0, v0, s0 = k.cpu().clone(), v.cpu().clone(), scores.cpu().clone()
    kept, _ = ctx.kv_evict(k, v, scores, lens, 64, sink=2, recent=16, kv_len_out=lens)
    assert lens.tolist() == [64, 64] and (scores[..., 64:] == 0).all()
    q = torch.randn((B, H, D), generator=g).half()
    got = ctx.attn_decode_shared(q.cuda(), None, None, k, v, lens)
    ks, vs = torch.zeros((B, 64, Hkv, D)).half(), torch.zeros((B, 64, Hkv, D)).half()
    for b, n in enumerate((200, 150)):
        for h in range(Hkv):
            rows = _kept64(s0[b, h].numpy(), n, 64, 2, 16)
            assert kept[b, h].tolist() == rows
            ks[b, :, h], vs[b, :, h] = k0[b, rows, h], v0[b, rows, h]
    want, A, ds, _, _ = _decode64(q, None, None, ks, vs, [64, 64], D ** -0.5)
    assert ((got.double().cpu() - want).abs() <= U["f16"] * want.abs() + (U["f16"] + 2 * ds + 2.0 ** -20) * A).all()


def test_decode_shared_writes_any_aligned_output(ctx):
    """Outputs two bytes off a 16-byte boundary, over the forms of the merge: the same values."""
    for B, H, Hkv, D, P, Tn in ((2, 8, 2, 64, 100, 30), (40, 32, 8, 128, 0, 50), (64, 32, 8, 128, 3000, 20)):
        g = _gen(B)
        q, k, v = (torch.randn(s, generator=g).half().cuda() for s in ((B, H, D), (B, Tn, Hkv, D), (B, Tn, Hkv, D)))
        kp, vp = (torch.randn((P, Hkv, D), generator=g).half().cuda() for _ in range(2)) if P else (None, None)
        want = ctx.attn_decode_shared(q, kp, vp, k, v)
        out = torch.zeros(B * H * D + 1, dtype=torch.float16, device="cuda")[1:].view(B, H, D)
        assert ctx.attn_decode_shared(q, kp, vp, k, v, out=out).data_ptr() == out.data_ptr()
        assert (out.float() - want.float()).abs().max() <= 2.0 ** -9  # one fp16 step below 4: another order of the pieces


def test_decode_shared_long_prefix_in_a_graph_and_back_to_back(ctx):
    """Three launches per call, the second beside the first: calls that follow one another share a workspace and do not disturb
    each other, whatever lies between them."""
    g = _gen(11)
    B, H, Hkv, D, P, Tn = 40, 32, 8, 128, 5000, 60
    calls = []
    for i in range(3):
        q, k, v = (torch.randn(s, generator=g).half().cuda() for s in ((B, H, D), (B, Tn, Hkv, D), (B, Tn, Hkv, D)))
        kp, vp = (torch.randn((P, Hkv, D), generator=g).half().cuda() for _ in range(2))
        lens = torch.randint(0, Tn + 1, (B,), generator=g, dtype=torch.int32).cuda()
        calls.append((q, kp, vp, k, v, lens))
    scores = [torch.zeros((B, Hkv, Tn), device="cuda") for _ in calls]
    want = []
    for c, s in zip(calls, scores):
        want.append(ctx.attn_decode_shared(*c, scores=s).clone())
        torch.cuda.synchronize()
    once = [s.clone() for s in scores]
    ws = ctx.SharedWorkspace(B, H, Hkv, D, rows=Tn)
    outs = [torch.empty_like(w) for w in want]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for c, s, o in zip(calls, scores, outs):
            ctx.attn_decode_shared(*c, scores=s, out=o, workspace=ws)
    for _ in range(4):
        graph.replay()
    for c, s, o in zip(calls, scores, outs):
        for _ in range(3):
            ctx.attn_decode_shared(*c, scores=s, out=o, workspace=ws)
    torch.cuda.synchronize()
    assert int(ws.status.item()) == 0
    for o, w, s, one in zip(outs, want, scores, once):
        assert torch.equal(o, w)
        assert (s - 8 * one).abs().max() <= 8 * 2.0 ** -22 * 4 * 8  # eight steps of weights of at most four each, added one by one


@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
@pytest.mark.parametrize("P, Tn", ((131072, 0), (131072, 300), (0, 4096)))
def test_fp32_outputs_of_long_sums_are_not_small(ctx, dtype, P, Tn):
    """Positive values: a bias of the sums shows. A matrix instruction may cut off up to one unit in the last place; a chain of them
    over one block has at most twelve. Additions of blocks and the probabilities' own roundings average out over rows and outputs,
    up to a common error of exp2, 2^-22. So the mean signed error is below 12 * 2^-23, that, and the few roundings of joining
    the pieces: 18 * 2^-23."""
    B, H, Hkv, D = 16, 8, 2, 128
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.zeros((B, H, D), dtype=dtype, device="cuda")
    q[:, :, 0] = 1
    k, kp = (torch.zeros(s, dtype=dtype, device="cuda") for s in ((B, Tn, Hkv, D), (P, Hkv, D)))
    v, vp = ((1 + torch.rand(s, generator=g, device="cuda")).to(dtype) for s in ((B, Tn, Hkv, D), (P, Hkv, D)))
    for x in (k, kp):
        x[..., 0] = (-2 * torch.rand(x.shape[:-1], generator=g, device="cuda")).to(dtype)
    out = ctx.attn_decode_shared(q, kp if P else None, vp if P else None, k, v, out_dtype=torch.float32, scale=1.0).double()
    w, wp = k[..., :1].double().exp(), kp[..., :1].double().exp()
    want = ((w * v.double()).sum(1) + (wp * vp.double()).sum(0)) / (w.sum(1) + wp.sum(0))
    want = want.repeat_interleave(H // Hkv, dim=1)
    assert abs(float(((out - want) / want).mean())) <= 18 * 2.0 ** -23


@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
@pytest.mark.parametrize("D", (64, 128))
def test_fp32_outputs_take_probabilities_in_full(ctx, dtype, D):
    """Two rows, one of score 0 and value 0, one of score -a and value 1: the output is p / (1 + p), p = exp(-a). Relative errors:
    of p 2^-22 (exp2) and 2^-22 (the scale's product), the sum 2^-24, the division 2^-23, three cut-off additions 2^-23 each, the
    joining of pieces 2^-21; together 6.25 * 2^-22. (A p of 16 bits would be off by up to 2^-17.)"""
    B, H = 4, 64
    a = ((1 + torch.arange(B * H, dtype=torch.float64)) / 128).to(dtype).cuda()  # up to 2, exact in either type
    q = torch.zeros((B, H, D), dtype=dtype, device="cuda")
    q[:, :, 0] = a.view(B, H)
    for prefix in (False, True):
        rows = 0 if prefix else 2
        k, v = torch.zeros((2, 1, D), dtype=dtype, device="cuda"), torch.zeros((2, 1, D), dtype=dtype, device="cuda")
        k[1, 0, 0] = -1
        v[1] = 1
        own = torch.zeros((B, 0, 1, D), dtype=dtype, device="cuda") if prefix else k[None].expand(B, -1, -1, -1).contiguous()
        own_v = own if prefix else v[None].expand(B, -1, -1, -1).contiguous()
        out = ctx.attn_decode_shared(q, k if prefix else None, v if prefix else None, own, own_v, out_dtype=torch.float32, scale=0.75).double()
        p = torch.exp(-0.75 * a.double()).view(B, H, 1)
        want = (p / (1 + p)).expand(B, H, D)
        assert own.shape[1] == rows
        assert float(((out - want) / want).abs().max()) <= 6.25 * 2.0 ** -22


def test_memory_of_a_call_belongs_to_its_stream(ctx):
    """Calls on a stream that is busy, without outputs or workspaces of the caller's: what the current stream allocates and writes in
    the meantime neither changes their results nor is changed by them."""
    g = _gen(5)
    B, H, Hkv, D, P, Tn = 8, 32, 8, 128, 3000, 700
    q, k, v = (torch.randn(s, generator=g).half().cuda() for s in ((B, H, D), (B, Tn, Hkv, D), (B, Tn, Hkv, D)))
    kp, vp = (torch.randn((P, Hkv, D), generator=g).half().cuda() for _ in range(2))
    zero = torch.zeros((B, Hkv, Tn), device="cuda")
    inv, _ = ctx.rope_frequencies(D, 10000.0)
    inv, pos, new = inv.cuda(), torch.arange(B, dtype=torch.int32, device="cuda"), torch.randn((B, Hkv, D), generator=g).half().cuda()

    def calls(stream):
        scores, cache = zero.clone(), [torch.zeros((B, 8, Hkv, D), dtype=torch.float16, device="cuda") for _ in range(2)]
        outs = [torch.zeros((B, 256, Hkv, D), dtype=torch.float16, device="cuda") for _ in range(2)] + [torch.zeros((B, Hkv, 256), device="cuda")]
        torch.cuda.synchronize()
        if stream is not None:
            with torch.cuda.stream(stream):
                torch.cuda._sleep(50_000_000)
        turned = ctx.rope_positions(q, new, new, *cache, pos, pos, inv_freq=inv, stream=stream)
        out = ctx.attn_decode_shared(turned, kp, vp, k, v, scores_out=scores, stream=stream)
        kept, lens = ctx.kv_evict(k, v, scores, None, 256, sink=4, recent=16, out=tuple(outs), stream=stream)
        return turned, out, scores, kept, lens, *outs, *cache  # (what the caller brought must live until the stream is through, the caches too)

    want = calls(None)
    side = torch.cuda.Stream()
    torch.cuda.empty_cache()
    sizes = (B * H * D * 2, B * Hkv * 256 * 4, B * 4, ctx.SharedWorkspace(B, H, Hkv, D, rows=Tn).nbytes)
    got = calls(side)
    assert not side.query()  # (still busy: nothing of it has run)
    others = [torch.full((n,), 7, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(4)]
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    for x in others:
        assert bool((x == 7).all())


@pytest.mark.parametrize("B, T, keep, Hkv, D", ((1, 1024, 256, 8, 128), (5, 700, 699, 4, 64), (2, 8192, 1000, 8, 128), (3, 300, 17, 2, 72),
                                                (1, 8192, 8192, 1, 64), (18, 129, 33, 8, 128)))
def test_evict_in_one_launch_or_two(ctx, B, T, keep, Hkv, D):
    """Small calls select and copy in one launch, except where the new lengths take the old ones' place: the same results."""
    g = _gen(T + keep)
    k, v = (torch.randn((B, T, Hkv, D), generator=g).half().cuda() for _ in range(2))
    scores = torch.randint(0, 50, (B, Hkv, T), generator=g).float().cuda()  # many ties
    lens = torch.randint(0, T + 1, (B,), generator=g, dtype=torch.int32).cuda()
    lens[0] = T
    results = []
    for alias in (False, True):
        outs = [torch.full((B, keep + 3, Hkv, D), 3.0, dtype=torch.float16, device="cuda") for _ in range(2)]
        outs.append(torch.full((B, Hkv, keep + 3), 3.0, device="cuda"))
        old = lens.clone()
        launches = ctx._b.load().attn_kernel_launch_count()
        kept, new = ctx.kv_evict(k, v, scores, old, keep, sink=4, recent=9, out=tuple(outs), kv_len_out=old if alias else None)
        assert ctx._b.load().attn_kernel_launch_count() - launches == (2 if alias else 1)
        assert torch.equal(new, lens.clamp(max=keep)) and (alias or torch.equal(old, lens))
        results.append((kept, new, *outs))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    kept = results[0][0]
    for b in range(B):  # and both copy what the list says
        n = min(int(lens[b]), keep)
        at = kept[b, :, :n].long()
        for h in range(Hkv):
            assert torch.equal(results[0][2][b, :n, h], k[b, at[h], h]) and torch.equal(results[0][3][b, :n, h], v[b, at[h], h])
            assert torch.equal(results[0][4][b, h, :n], scores[b, h, at[h]])
        assert bool((kept[b, :, n:] == -1).all()) and bool((results[0][4][b, :, n:] == 0).all()) and bool((results[0][2][b, n:] == 3).all())
