"""8-bit integer operators in the forms that few sizes reach: pairs of CTAs over a whole vocabulary and over many steps of the inner
dimension, rings of rows in wider buffers, weights that are rewritten between products, operands that lie between each other."""
import pytest
import torch

from test_int8_gpu import DEV, EPS, T, _eight_bits, _gen, _rand, check_product, i8, norm_of, scale_tolerance, whole_numbers  # noqa: F401

pytestmark = pytest.mark.gpu


def _operands(i8, m, k, rows, seed):  # noqa: F811
    g = _gen(seed)
    return (_eight_bits(i8, g, m, k), torch.rand(m, generator=g, device=DEV) * 0.02, _eight_bits(i8, g, rows, k, lowest=-128),
            torch.rand(rows, generator=g, device=DEV) * 2e-3 * k ** -0.5)


@pytest.mark.parametrize("m,k,n", [(33, 300, 76000), (61, 1011, 75905), (64, 2100, 75780), (40, 128, 80001), (2, 16, 8388700)])
@pytest.mark.parametrize("swiglu", [False, True])
def test_a_whole_vocabulary_of_channels(i8, m, k, n, swiglu):  # noqa: F811
    """33 to 64 tokens times more channels than four tiles for each SM (or more tiles than a grid's third dimension has): pairs with
    64 tokens a tile, a few hundred tiles for 74 pairs, the last ones cut off in both directions."""
    a, a_scale, w, w_scale = _operands(i8, m, k, 2 * n if swiglu else n, m + k + n)
    for dtype in T.values():
        check_product(i8, a, a_scale, w, w_scale, swiglu, dtype)


@pytest.mark.parametrize("m,k,n,swiglu", [(2000, 4096, 1500, False), (4500, 2000, 1500, False), (1500, 4096, 1500, True), (9000, 1300, 700, True),
                                          (1003, 14336, 4096, False), (300, 6000, 300, True), (700, 5003, 900, False)])
def test_many_steps_through_a_pairs_ring(i8, m, k, n, swiglu):  # noqa: F811
    """Tiles of 256 and of 128 tokens whose inner dimension fills the ring again and again, several tiles a pair."""
    a, a_scale, w, w_scale = _operands(i8, m, k, 2 * n if swiglu else n, m + k + n)
    for dtype in T.values():
        check_product(i8, a, a_scale, w, w_scale, swiglu, dtype)


RINGS = [("f32", None, 6912), ("f16", None, 14336), ("bf16", None, 13832), ("f32", "f32", 8960), ("f32", "bf16", 11008), ("bf16", "f32", 16384),
         ("f16", "f16", 16392), ("bf16", "none", 16384), ("f32", "none", 9216)]


@pytest.mark.parametrize("rows", [299, 601])
@pytest.mark.parametrize("shift", [16, 4, 1])
@pytest.mark.parametrize("dtype,delta_type,dim", RINGS)
def test_rings_of_rows_in_wider_buffers(i8, rows, shift, dtype, delta_type, dim):  # noqa: F811
    """More rows than two for each SM, long ones, between others' values (shift 16: as bulk copies take them; else as 16-byte accesses do
    not). delta_type None: quantisation; "none": the norm by itself. Neighbours of what is written stay as they were."""
    g = _gen(rows + shift + dim)
    big = _rand(g, rows, dim + 48, dtype=T[dtype])
    x, before = big[:, shift:shift + dim], big.clone()
    store = torch.full((rows, (dim + 15) // 16 * 16 + 32), 77, dtype=torch.int8, device=DEV)
    scale = torch.full((rows + 2,), -1.0, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    kw = dict(out=store[:, 16:16 + dim], scale=scale[1:rows + 1], status=status)
    if delta_type is None:
        q, s = i8.quantize_i8(x, **kw)
        z, want, relative = x.float(), x.double().abs().amax(1) / 127.0, 2.0 ** -24
    else:
        weight = 1.0 + 0.1 * _rand(g, dim)
        delta = None if delta_type == "none" else _rand(g, rows, dim + 40, dtype=T[delta_type])[:, 24:24 + dim]
        h, z, want = norm_of(x, weight, delta)
        relative = scale_tolerance(dim)
        q, s = i8.rmsnorm_i8(x, weight, EPS, delta=delta, **kw)  # in place
        if delta is not None:
            before[:, shift:shift + dim] = h.to(T[dtype])
    torch.cuda.synchronize()
    assert torch.equal(q, whole_numbers(z)) and ((s.double() - want).abs() <= want * relative).all()
    assert torch.equal(big, before) and int(status.item()) == 0
    assert (store[:, :16] == 77).all() and (store[:, 16 + dim:] == 77).all() and scale[0] == -1 and scale[-1] == -1


@pytest.mark.parametrize("dtype,dim", [("f32", 8960), ("f16", 16384), ("bf16", 14336)])
def test_special_rows_in_a_ring(i8, dtype, dim):  # noqa: F811
    """Zeros, NaN and infinities leave the rows before and behind them in the same slots alone."""
    x = _rand(_gen(dim), 1000, dim, dtype=T[dtype])
    x[5::97] = 0
    x[7::101, dim - 1] = float("nan")
    x[11::103, 3] = -float("inf")
    bad = ~torch.isfinite(x).all(1)
    q, scale = i8.quantize_i8(x)
    qn, sn = i8.rmsnorm_i8(x, torch.ones(dim, device=DEV), EPS)
    torch.cuda.synchronize()
    want = whole_numbers(x[~bad].float())
    for got, s in ((q, scale), (qn, sn)):
        assert torch.equal(got[~bad], want) and (got[bad] == 0).all() and torch.equal(torch.isnan(s), bad)
        assert torch.equal(s == 0, (x == 0).all(1))


@pytest.mark.parametrize("m,k,n,swiglu", [(1, 4096, 4096, False), (9, 5000, 640, True), (64, 4096, 200, True), (40, 300, 76000, False), (130, 6000, 300, False),
                                          (130, 6000, 300, True), (500, 1000, 1200, True), (1500, 2048, 1500, True)])
@pytest.mark.parametrize("early", [False, True])
def test_weights_that_are_rewritten_between_products(i8, m, k, n, swiglu, early):  # noqa: F811
    """Each product reads what the kernel right in front of it has just written over the last product's weights; what was brought to L2
    ahead of that may not be what is multiplied. With ``early`` the weights are complete and the rows are rewritten instead."""
    g, steps = _gen(m + n + k), 10
    count = 2 * n if swiglu else n
    sources = [_rand(g, count, k, dtype=torch.bfloat16) for _ in range(2)]
    x = [_rand(g, m, k) for _ in range(steps)]
    w, ws, a, s = i8.rows_i8(count, k), torch.empty(count, device=DEV), i8.rows_i8(m, k), torch.empty(m, device=DEV)
    i8.quantize_i8(sources[0], out=w, scale=ws)
    i8.quantize_i8(x[0], out=a, scale=s)
    outs = [torch.zeros((m, n), device=DEV) for _ in range(steps)]

    def run(wait=lambda: None):
        for i, out in enumerate(outs):
            if early:
                i8.quantize_i8(x[i], out=a, scale=s)
            else:
                i8.quantize_i8(sources[i % 2], out=w, scale=ws)
            wait()
            i8.gemm_i8(a, s, w, ws, out=out, swiglu=swiglu, w_early=early)
            wait()

    torch.cuda.synchronize()
    run(torch.cuda.synchronize)
    want = [t.clone() for t in outs]
    assert early or not torch.equal(want[0], want[1])
    torch.cuda.synchronize()
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


@pytest.mark.parametrize("rows,dim", [(5, 96), (400, 9216)])
def test_rows_between_each_other(i8, rows, dim):  # noqa: F811
    """x, delta, x_out and q side by side in the rows of one buffer share no byte: taken, and right."""
    g = _gen(rows)
    big = _rand(g, rows, 4 * dim)
    x, delta, x_out = big[:, :dim], big[:, dim:2 * dim], big[:, 2 * dim:3 * dim]
    q_out = big[:, 3 * dim:].view(torch.int8)[:, :dim]
    weight = 1.0 + 0.1 * _rand(g, dim)
    before = big.clone()
    h, z, want = norm_of(x, weight, delta)
    q, s = i8.rmsnorm_i8(x, weight, EPS, delta=delta, x_out=x_out, out=q_out)
    torch.cuda.synchronize()
    assert torch.equal(q, whole_numbers(z)) and ((s.double() - want).abs() <= want * scale_tolerance(dim)).all()
    assert torch.equal(x_out, h) and torch.equal(big[:, :2 * dim], before[:, :2 * dim])
    assert torch.equal(big[:, 3 * dim:].view(torch.int8)[:, dim:], before[:, 3 * dim:].view(torch.int8)[:, dim:])


@pytest.mark.parametrize("m,k,n", [(3, 160, 40), (300, 1000, 200)])
def test_a_products_rows_between_its_operands(i8, m, k, n):  # noqa: F811
    """The output's rows behind the tokens' in one buffer."""
    g = _gen(m)
    wide = (k + 15) // 16 * 16 + 4 * n
    store = torch.randint(-128, 128, (m, (wide + 15) // 16 * 16), generator=g, device=DEV, dtype=torch.int8)
    a, out = store[:, :k], store[:, (k + 15) // 16 * 16:][:, :4 * n].view(torch.float32)
    before = store.clone()
    w, one = _eight_bits(i8, g, n, k), torch.ones(max(m, n), device=DEV)
    check_product(i8, a, one[:m], w, one[:n], False, torch.float32, out=out)
    assert torch.equal(store[:, :(k + 15) // 16 * 16], before[:, :(k + 15) // 16 * 16])
