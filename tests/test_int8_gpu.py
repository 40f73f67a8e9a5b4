"""8-bit integer operators against plain implementations. q and sums are whole numbers: they have to be equal. Everything else is held
to the roundings that it goes through."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"
EPS = 1e-5


@pytest.fixture(scope="module")
def i8(built_lib, pkg):
    from llm_infer_b200 import int8
    return int8


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rand(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=DEV).to(dtype)


def whole_numbers(z):
    """The definition of q, operation by operation in fp32 (z fp32)."""
    top = z.abs().amax(1, keepdim=True)
    inverse = torch.where(top > 0, torch.full_like(top, 127.0) / top, torch.zeros_like(top))
    return torch.round(z * inverse).to(torch.int8)


def norm_of(x, weight, delta, eps=EPS):
    """h, z in fp32 as defined, and the scales in 64 bits."""
    h = x.float() if delta is None else x.float() + delta.float()
    z = h * weight
    h64 = h.double()
    factor = 1.0 / torch.sqrt((h64 * h64).mean(1) + eps)
    return h, z, z.double().abs().amax(1) * factor / 127.0


def scale_tolerance(dim):
    """Relative: the sum of squares of a row is added in runs of dim / 1024 + 32 at most and two trees of 5 levels, each addition off by
    2^-24; half of that on its root. Mean, eps, root, reciprocal, product and the division by 127: 2^-24 each, half of it ahead of the root."""
    return 2.0 ** -24 * ((dim / 1024 + 32 + 10) / 2 + 6)


ROWS = [(1, 1), (1, 4096), (2, 16), (3, 7), (5, 31), (4, 128), (7, 129), (33, 64), (64, 512), (9, 1000), (61, 5003), (2, 16384), (3, 16388),
        (2, 28672), (1, 32768), (3, 33000), (1, 70001), (300, 1024), (1003, 96), (301, 8192), (700, 14336),
        (450, 16384), (299, 28672)]


@pytest.mark.parametrize("rows,dim", ROWS)
@pytest.mark.parametrize("dtype", list(T))
def test_quantize_gives_the_defined_whole_numbers(i8, rows, dim, dtype):
    x = _rand(_gen(rows * 7 + dim), rows, dim, dtype=T[dtype])
    q, scale = i8.quantize_i8(x)
    torch.cuda.synchronize()
    assert q.shape == x.shape and torch.equal(q, whole_numbers(x.float()))
    want = x.double().abs().amax(1) / 127.0
    assert ((scale.double() - want).abs() <= want * 2.0 ** -24).all()  # one division


@pytest.mark.parametrize("rows,dim", ROWS)
@pytest.mark.parametrize("dtype,delta_type", [("f32", None), ("f32", "f32"), ("f32", "f16"), ("f16", "f16"), ("bf16", "f32"), ("bf16", "bf16"),
                                              ("f16", None), ("bf16", "f16"), ("f16", "bf16"), ("f32", "bf16"), ("bf16", None), ("f16", "f32")])
def test_norm_gives_the_defined_whole_numbers_and_scales(i8, rows, dim, dtype, delta_type):
    g = _gen(rows * 11 + dim)
    x, weight = _rand(g, rows, dim, dtype=T[dtype]), 1.0 + 0.1 * _rand(g, dim)
    delta = None if delta_type is None else _rand(g, rows, dim, dtype=T[delta_type])
    before = x.clone()
    x_out = None if delta is None else torch.empty_like(x)
    q, scale = i8.rmsnorm_i8(x, weight, EPS, delta=delta, x_out=x_out)
    torch.cuda.synchronize()
    h, z, want = norm_of(before, weight, delta)
    assert torch.equal(q, whole_numbers(z))
    assert ((scale.double() - want).abs() <= want * scale_tolerance(dim)).all()
    assert torch.equal(x, before)
    if delta is not None:
        assert torch.equal(x_out, h.to(T[dtype]))
        q2, scale2 = i8.rmsnorm_i8(x, weight, EPS, delta=delta)  # in place
        torch.cuda.synchronize()
        assert torch.equal(x, x_out) and torch.equal(q2, q) and torch.equal(scale2, scale)


@pytest.mark.parametrize("dim", [31, 256, 5003, 16400, 40000])
@pytest.mark.parametrize("dtype", list(T))
def test_rows_of_wider_buffers(i8, dim, dtype):
    """Strided x, delta, x_out and q: neighbours of the rows stay as they were. Offsets that 16-byte accesses cannot take as well."""
    g, rows = _gen(dim), 6
    for shift, wide in ((0, dim + 48 - dim % 16), (1, dim + 3), (8, 2 * dim + 16 - 2 * dim % 16)):
        big = _rand(g, rows + 1, wide, dtype=T[dtype])
        if shift + dim > wide:
            continue
        x = big[:rows, shift:shift + dim]
        delta = _rand(g, rows, wide, dtype=T[dtype])[:, wide - dim:]
        store = torch.full((rows, (dim + 15) // 16 * 16 + 32), 77, dtype=torch.int8, device=DEV)
        scale = torch.full((rows + 2,), -1.0, device=DEV)
        weight = 1.0 + 0.1 * _rand(g, dim + 1)[shift % 2:dim + shift % 2]
        before = big.clone()
        h, z, want = norm_of(x, weight, delta)
        q, s = i8.rmsnorm_i8(x, weight, EPS, delta=delta, out=store[:, 16:16 + dim], scale=scale[1:rows + 1])
        torch.cuda.synchronize()
        assert torch.equal(q, whole_numbers(z)) and ((s.double() - want).abs() <= want * scale_tolerance(dim)).all()
        before[:rows, shift:shift + dim] = h.to(T[dtype])
        assert torch.equal(big, before)
        assert (store[:, :16] == 77).all() and (store[:, 16 + dim:] == 77).all()
        assert scale[0] == -1 and scale[-1] == -1


@pytest.mark.parametrize("dim", [5, 300, 4096, 33000])
@pytest.mark.parametrize("dtype", list(T))
def test_special_rows(i8, dim, dtype):
    """Zeros, NaN, infinities, the smallest and the largest values: each row by itself."""
    x = _rand(_gen(3), 8, dim, dtype=T[dtype])
    tiny, huge = torch.finfo(T[dtype]).smallest_normal / 4, torch.finfo(T[dtype]).max
    x[0] = 0
    x[1, dim // 2] = float("nan")
    x[2, dim - 1] = float("inf")
    x[3, 0] = -float("inf")
    x[4] = x[4].sign() * tiny
    x[5, dim // 3] = huge
    q, scale = i8.quantize_i8(x)
    torch.cuda.synchronize()
    assert (q[:4] == 0).all() and scale[0] == 0 and torch.isnan(scale[1:4]).all()
    assert torch.equal(q[4].float(), 127.0 * x[4].sign().float())
    want = x[4].double().abs().amax() / 127.0
    assert abs(float(scale[4]) - float(want)) <= float(want) * 2.0 ** -24 + 2.0 ** -150  # (below the normal numbers: half a step)
    assert torch.equal(q[5:], whole_numbers(x[5:].float()))
    weight = torch.ones(dim, device=DEV)
    delta = torch.zeros_like(x)
    q, scale = i8.rmsnorm_i8(x, weight, EPS, delta=delta, x_out=torch.empty_like(x))
    torch.cuda.synchronize()
    assert (q[:4] == 0).all() and scale[0] == 0 and torch.isnan(scale[1:4]).all()
    if dtype == "f16":  # the squares fit fp32
        assert torch.isfinite(scale[5]) and torch.equal(q[5:], whole_numbers(x[5:].float()))
    else:
        assert torch.isnan(scale[5]) and (q[5] == 0).all()  # ... and here their sum does not
    assert torch.isfinite(scale[6:]).all()


def product(a, a_scale, w, w_scale, swiglu, dtype):
    """The definition: the exact sum, rounded to fp32, times the channel's and the token's scale, each product rounded. Second: a bound
    on how far the result may be from the first. Without SwiGLU none: the same operations. With it: exp is good to two units (2^-22)
    and so is the quotient, the sum and the product round once each (2^-24), the result once to its type."""
    sums = (a.double() @ w.double().t())
    y = sums.float() * w_scale * a_scale[:, None]
    if not swiglu:
        return y.to(dtype), torch.zeros_like(y, dtype=torch.float64)
    n = w.shape[0] // 2
    gate, up = y[:, :n].double(), y[:, n:].double()
    want = gate / (1.0 + torch.exp(-gate)) * up
    step = 2.0 ** -24 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    # (below the type's smallest normal number, 2^-14 in fp16, its values are a fixed distance apart, 2^-24: half of that is the rounding)
    least = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    return want, want.abs() * (2 * 2.0 ** -22 + 2 * 2.0 ** -24 + step) * 1.01 + least + 1e-37


def _eight_bits(i8, g, rows, k, lowest=-127):
    q = i8.rows_i8(rows, k)
    q.copy_(torch.randint(lowest, 128, (rows, k), generator=g, device=DEV, dtype=torch.int8))
    return q


def check_product(i8, a, a_scale, w, w_scale, swiglu, dtype, **kw):
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = i8.gemm_i8(a, a_scale, w, w_scale, swiglu=swiglu, out_dtype=dtype, status=status, **kw)
    torch.cuda.synchronize()
    assert int(status.item()) == 0
    want, bound = product(a, a_scale, w, w_scale, swiglu, dtype)
    if swiglu:
        assert ((out.double() - want).abs() <= bound).all()
    else:
        assert torch.equal(out, want)
    return out


SHAPES = [(1, 1, 1), (1, 16, 1), (1, 128, 128), (1, 4096, 6144), (2, 129, 127), (3, 33, 500), (7, 4096, 4096), (8, 14336, 1024), (15, 1000, 129),
          (16, 2048, 257), (17, 2048, 256), (31, 144, 1003), (32, 640, 640), (33, 640, 640), (61, 4096, 2049), (64, 4096, 4096), (65, 100, 300),
          (100, 5003, 777), (128, 1024, 1024), (129, 1024, 4100), (203, 1011, 4099), (256, 4096, 512), (257, 512, 513), (300, 4096, 4096),
          (511, 333, 1000), (1003, 1536, 1111), (1024, 128, 2048), (2048, 256, 300), (700, 14336, 1024), (4097, 1, 3), (3000, 64, 4096)]


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("swiglu", [False, True])
def test_products_are_the_exact_sums_scaled(i8, m, k, n, swiglu):
    g = _gen(m * 131 + k * 17 + n)
    rows = 2 * n if swiglu else n
    a, w = _eight_bits(i8, g, m, k), _eight_bits(i8, g, rows, k, lowest=-128)
    a_scale, w_scale = torch.rand(m, generator=g, device=DEV) * 0.02, torch.rand(rows, generator=g, device=DEV) * 2e-3 / math.sqrt(k)
    for dtype in T.values():
        check_product(i8, a, a_scale, w, w_scale, swiglu, dtype)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_longest_sums_of_largest_values(i8, m):
    """k = 131071 products of -128 and -127 or 127: up to 2^31 - 2 million, in one slice's or in several slices' sums."""
    k, n = i8.MAX_K, 130
    a, w = i8.rows_i8(m, k), i8.rows_i8(n, k)
    a.fill_(-128), w.fill_(-128)
    a[m // 2] = 127
    w[77] = 127
    one = torch.ones(max(m, n), device=DEV)
    out = check_product(i8, a, one[:m], w, one[:n], False, torch.float32)
    assert float(out[m // 2, 0]) == float(torch.tensor(-127.0 * 128 * k, dtype=torch.float32))


@pytest.mark.parametrize("m,k,n", [(1, 300, 200), (20, 1000, 333), (150, 260, 500), (600, 700, 900)])
@pytest.mark.parametrize("swiglu", [False, True])
def test_strided_operands_and_what_lies_beside_them(i8, m, k, n, swiglu):
    """Rows of wider buffers whose other bytes are garbage; rows and columns of the output's buffer beside it stay as they were."""
    g = _gen(m + k + n)
    rows = 2 * n if swiglu else n
    wide = (k + 15) // 16 * 16 + 48
    big_a = torch.randint(-128, 128, (m + 2, wide), generator=g, device=DEV, dtype=torch.int8)
    big_w = torch.randint(-128, 128, (rows + 2, wide), generator=g, device=DEV, dtype=torch.int8)
    a, w = big_a[1:m + 1, 16:16 + k], big_w[1:rows + 1, 32:32 + k]
    a_scale, w_scale = torch.rand(m + 2, generator=g, device=DEV)[1:m + 1] * 0.01, torch.rand(rows + 1, generator=g, device=DEV)[1:] * 1e-3
    for dtype in T.values():
        store = torch.full((m + 2, n + 7), 55.0, dtype=dtype, device=DEV)
        check_product(i8, a, a_scale, w, w_scale, swiglu, dtype, out=store[1:m + 1, 3:3 + n])
        assert (store[0] == 55).all() and (store[-1] == 55).all() and (store[:, :3] == 55).all() and (store[:, 3 + n:] == 55).all()


def test_a_token_has_the_same_bits_in_every_batch(i8):
    g, k, n = _gen(5), 4096, 1500
    w, w_scale = _eight_bits(i8, g, 2 * n, k), torch.rand(2 * n, generator=g, device=DEV) * 1e-3
    a, a_scale = _eight_bits(i8, g, 2000, k), torch.rand(2000, generator=g, device=DEV) * 0.01
    for swiglu in (False, True):
        whole = i8.gemm_i8(a, a_scale, w, w_scale, swiglu=swiglu)
        for lo, hi in ((0, 1), (3, 11), (100, 140), (64, 164), (500, 1100)):
            assert torch.equal(i8.gemm_i8(a[lo:hi], a_scale[lo:hi], w, w_scale, swiglu=swiglu), whole[lo:hi])


@pytest.mark.parametrize("m", [2, 50, 400])
def test_scales_that_are_not_numbers_stay_in_their_token_or_channel(i8, m):
    g, k, n = _gen(6), 512, 384
    a, w = _eight_bits(i8, g, m, k), _eight_bits(i8, g, n, k)
    a_scale, w_scale = torch.rand(m, generator=g, device=DEV) + 0.1, torch.rand(n, generator=g, device=DEV) + 0.1
    a_scale[1], w_scale[200] = float("nan"), float("inf")
    out = i8.gemm_i8(a, a_scale, w, w_scale)
    torch.cuda.synchronize()
    want = (a.double() @ w.double().t()).float() * w_scale * a_scale[:, None]
    assert torch.isnan(out[1]).all() and torch.equal(torch.isnan(out), torch.isnan(want))
    assert torch.equal(out.nan_to_num(), want.nan_to_num())


def _layer(i8, m, dim, hidden, g):
    """What one pass through the linear part of a layer needs."""
    w13, s13 = i8.quantize_i8(_rand(g, 2 * hidden, dim) * dim ** -0.5)
    w2, s2 = i8.quantize_i8(_rand(g, dim, hidden) * hidden ** -0.5)
    return dict(x=_rand(g, m, dim), d=_rand(g, m, dim), weight=1.0 + 0.1 * _rand(g, dim), w13=w13, s13=s13, w2=w2, s2=s2)


def _run_layer(i8, s, wait=lambda: None, stream=None):
    x = torch.empty_like(s["x"])
    wait()
    q, scale = i8.rmsnorm_i8(s["x"], s["weight"], EPS, delta=s["d"], x_out=x, stream=stream)
    wait()
    h = i8.gemm_i8(q, scale, s["w13"], s["s13"], swiglu=True, out_dtype=torch.bfloat16, stream=stream)
    wait()
    q2, scale2 = i8.quantize_i8(h, stream=stream)
    wait()
    y = i8.gemm_i8(q2, scale2, s["w2"], s["s2"], stream=stream)
    wait()
    return x, q, scale, h, q2, scale2, y


@pytest.mark.parametrize("m,dim,hidden", [(1, 4096, 14336), (5, 1000, 2051), (77, 640, 1999), (600, 1024, 2048)])
def test_a_layers_calls_one_behind_the_other(i8, m, dim, hidden):
    """Norm, projection with SwiGLU, quantisation, projection: launched without a wait between them, on another stream, and in a
    graph that is replayed, each call right behind the one that writes its operands, the results are those of calls that are waited for."""
    s = _layer(i8, m, dim, hidden, _gen(m + dim))
    torch.cuda.synchronize()
    want = [t.clone() for t in _run_layer(i8, s, torch.cuda.synchronize)]
    h, z, scale = norm_of(s["x"], s["weight"], s["d"])
    assert torch.equal(want[0], h) and torch.equal(want[1], whole_numbers(z))
    up, bound = product(want[1], want[2], s["w13"], s["s13"], True, torch.bfloat16)
    assert ((want[3].double() - up).abs() <= bound).all()
    assert torch.equal(want[4], whole_numbers(want[3].float()))
    assert torch.equal(want[6], product(want[4], want[5], s["w2"], s["s2"], False, torch.float32)[0])
    # and the whole is near the layer in 64 bits: rows of 127 steps either side, weights too
    y64 = norm_of(s["x"], s["weight"], s["d"])[1].double() / torch.sqrt((h.double() ** 2).mean(1, keepdim=True) + EPS)
    gate, up64 = (y64 @ (s["w13"].double() * s["s13"].double()[:, None]).t()).split(hidden, 1)
    far = (gate * torch.sigmoid(gate) * up64) @ (s["w2"].double() * s["s2"].double()[:, None]).t()
    assert float((want[6].double() - far).norm() / far.norm()) < 0.05
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(_run_layer(i8, s), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = _run_layer(i8, s, stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = _run_layer(i8, s)
        graphs.append((graph, outs))
    for _ in range(3):
        for graph, outs in graphs:
            for t in outs:
                t.zero_()
            graph.replay()
    torch.cuda.synchronize()
    for _, outs in graphs:
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("m,k,n,swiglu", [(1, 4096, 4096, False), (1, 100, 130, False), (9, 5000, 640, True), (40, 2048, 3000, False), (64, 4096, 200, True),
                                          (130, 6000, 300, False), (500, 1000, 1200, False)])
def test_weights_requested_early(i8, m, k, n, swiglu):
    """w_early: weights that nothing writes are read while the kernels in front still run; what those write is waited for. Chains of
    quantisation and product, each reading what the one before it wrote, in a row and in a graph."""
    g, steps = _gen(m + n), 12
    rows = 2 * n if swiglu else n
    w, ws = i8.quantize_i8(_rand(g, rows, k))
    x = [_rand(g, m, k) for _ in range(steps)]
    q, s = i8.rows_i8(m, k), torch.empty(m, device=DEV)
    outs = [torch.zeros((m, n), device=DEV) for _ in range(steps)]
    torch.cuda.synchronize()
    want = [i8.gemm_i8(*i8.quantize_i8(y), w, ws, swiglu=swiglu) for y in x]
    torch.cuda.synchronize()

    def run():
        for y, out in zip(x, outs):
            i8.quantize_i8(y, out=q, scale=s)
            i8.gemm_i8(q, s, w, ws, out=out, swiglu=swiglu, w_early=True)

    run()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for _ in range(3):
        for out in outs:
            out.zero_()
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_offsets_that_pass_32_bits(i8):
    """More than 2^32 values in an output, and in the rows that are quantised; rows of an operand further than 2^32 bytes behind its first."""
    g = _gen(12)
    m, n, k = 66000, 66000, 16
    a, w = _eight_bits(i8, g, m, k), _eight_bits(i8, g, n, k)
    one = torch.ones(m, device=DEV)
    out = i8.gemm_i8(a, one, w, one, out_dtype=torch.float16)
    for t in (0, 1, 32767, 65076, 65999):
        assert torch.equal(out[t], (a[t:t + 1].double() @ w.double().t()).half()[0])
    del out
    rows, dim = 140000, 32768
    x = torch.empty((rows, dim), dtype=torch.float16, device=DEV)
    for lo in range(0, rows, 20000):
        x[lo:lo + 20000] = _rand(g, min(20000, rows - lo), dim, dtype=torch.float16)
    q, scale = i8.quantize_i8(x)
    for t in (0, 131071, 131072, 139999):
        assert torch.equal(q[t:t + 1], whole_numbers(x[t:t + 1].float())) and abs(float(scale[t]) * 127 / float(x[t].abs().max()) - 1) < 2.0 ** -22
    # the last rows as an operand of the product, reached from the first row's address
    far = q[::1000, :2048]
    assert far.stride(0) * (far.shape[0] - 1) > 2 ** 32
    for m in (far.shape[0], 3):
        b, bs = far[-m:], scale[::1000][-m:].contiguous()
        got = i8.gemm_i8(far, scale[::1000].contiguous(), b, bs)
        assert torch.equal(got, (far.double() @ b.double().t()).float() * bs * scale[::1000][:, None])
    torch.cuda.synchronize()


def test_a_matrix_with_itself(i8):
    q, s = i8.quantize_i8(_rand(_gen(13), 200, 1000))
    out = i8.gemm_i8(q, s, q, s)
    assert torch.equal(out, (q.double() @ q.double().t()).float() * s * s[:, None])


def test_empty_calls_and_refusals(i8):
    g = _gen(9)
    x, weight = _rand(g, 4, 64), torch.ones(64, device=DEV)
    q, s = i8.quantize_i8(x)
    w, ws = i8.quantize_i8(_rand(g, 6, 64))
    e, es = i8.quantize_i8(x[:0])
    assert e.shape == (0, 64) and es.shape == (0,)
    assert i8.gemm_i8(e, es, w, ws).shape == (0, 6)
    assert i8.gemm_i8(q, s, w[:0], ws[:0]).shape == (4, 0)
    bad = [
        lambda: i8.quantize_i8(x[0]), lambda: i8.quantize_i8(x.double()), lambda: i8.quantize_i8(x[:, ::2]), lambda: i8.quantize_i8(x[:, :0]),
        lambda: i8.quantize_i8(x[:1].expand(4, 64)), lambda: i8.quantize_i8(x, out=torch.empty((4, 60), dtype=torch.int8, device=DEV)),
        lambda: i8.quantize_i8(x[:, :60].contiguous(), out=torch.empty((4, 60), dtype=torch.int8, device=DEV)),
        lambda: i8.quantize_i8(x, out=torch.empty((4, 64), dtype=torch.uint8, device=DEV)),
        lambda: i8.quantize_i8(x, scale=torch.empty(5, device=DEV)), lambda: i8.quantize_i8(x, scale=x[:, 0]),
        lambda: i8.rmsnorm_i8(x, weight[:63], EPS), lambda: i8.rmsnorm_i8(x, weight.half(), EPS), lambda: i8.rmsnorm_i8(x, weight, 0.0),
        lambda: i8.rmsnorm_i8(x, weight, EPS, x_out=x), lambda: i8.rmsnorm_i8(x, weight, EPS, delta=x[:3]),
        lambda: i8.rmsnorm_i8(x, weight, EPS, delta=x, x_out=x), lambda: i8.rmsnorm_i8(x, weight, EPS, delta=x.clone(), x_out=x.half()),
        lambda: i8.rmsnorm_i8(x, weight.cpu(), EPS),
        lambda: i8.gemm_i8(q, s, w[:, :32], ws), lambda: i8.gemm_i8(q, s[:3], w, ws), lambda: i8.gemm_i8(q, s, w, ws[:3]),
        lambda: i8.gemm_i8(q.float(), s, w, ws), lambda: i8.gemm_i8(q, s, w[:5], ws[:5], swiglu=True),
        lambda: i8.gemm_i8(q, s, w, ws, out_dtype=torch.float64), lambda: i8.gemm_i8(q, s, w, ws, out=torch.empty((4, 5), device=DEV)),
        lambda: i8.gemm_i8(q[:, :40], s, torch.zeros((6, 40), dtype=torch.int8, device=DEV), ws),
        lambda: i8.gemm_i8(q.cpu(), s, w, ws), lambda: i8.gemm_i8(q[:, 8:40], s, w[:, 8:40], ws),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, TypeError, i8._b.AttnError)):
            call()
            pytest.fail(f"call {i} was taken")
    torch.cuda.synchronize()
