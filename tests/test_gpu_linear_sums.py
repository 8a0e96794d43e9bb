"""Long sums of spmm_cpp.linear: many rows in the weight gradient, many columns in the product, on operands of one sign, where what an accumulator
truncates adds up, against float64.  Needs a GPU.

An accumulation into the tensor cores' accumulator is off by up to three steps (2^-23) of the running sum, on average over a sum that grows evenly three halves of a step of
the whole.  Chains of them end, and their sums are added in fp32: after 512 (fp16), 2,048 (bf16) and 128 (fp32, of 8 columns) accumulations, CHAIN below.  The result
rounds by half a step of its type, evenly in both directions: over n elements the mean of that is zero within 6 half steps / sqrt(3 n)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
CHAIN = {torch.float32: 128 * 1.5 * 2.0 ** -23, torch.bfloat16: 2048 * 1.5 * 2.0 ** -23, torch.float16: 512 * 1.5 * 2.0 ** -23}


def _positive(gen, *shape, dtype):
    return torch.rand(shape, device='cuda', generator=gen, dtype=torch.float32).to(dtype)


def _check(got, want, dtype, added=0.0):
    off = got.double() / want - 1
    bound = CHAIN[dtype] + added
    assert float(off.abs().max()) <= HALF[dtype] + bound, float(off.abs().max())
    # Sums of 65,536 terms of one sign differ by 0.3 % (the product of two even numbers of [0, 1) has a spread of 0.88 of its mean, 65,536 of them a 256th of that), about as much as half a step of bf16: their roundings are not even, and
    # their mean is not zero but a number that the exact values tell, moved by as much as the chains may move them (in quarters).
    uneven = max(float((((want * (1 - bound * i / 4)).to(dtype).double() - want * (1 - bound * i / 4)) / want).mean().abs()) for i in range(5))
    assert float(off.mean().abs()) <= bound + uneven + 6 * HALF[dtype] / (3 * off.numel()) ** 0.5, float(off.mean())


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('M,K,N,act', [(300_000, 264, 2304, None), (131_072, 2304, 2304, None), (70_001, 64, 19_200, 'relu'), (70_001, 40, 19_208, 'silu'), (100_003, 72, 200, None),
                                       (9_000, 2304, 2312, None)])
def test_weight_gradients_of_many_rows(M, K, N, act, dtype):
    """Ranges of one chain and of several, one range and many, dz as it comes and made on the way."""
    import spmm_cpp
    gen = torch.Generator(device='cuda').manual_seed(M + N)
    x, w = _positive(gen, M, K, dtype=dtype), (_positive(gen, K, N, dtype=dtype) / K).requires_grad_()
    dy = _positive(gen, M, N, dtype=dtype) * (64 / M)
    y = spmm_cpp.linear(x, w, activation=act)
    dw, = torch.autograd.grad(y, w, dy)
    columns = torch.tensor([0, 1, 17, N // 2, N - 9, N - 1, *range(N - 40, N - 12)], device='cuda')
    dz = dy[:, columns].double()
    if act == 'silu':                                              # with the z that the kernel keeps, rounded to the type, and dz rounded
        z = (x.double() @ w.detach()[:, columns].double()).to(dtype).double()
        s = torch.sigmoid(z)
        dz = dz * s * (1 + z * (1 - s))
    rows = torch.cat([torch.arange(min(K, 48), device='cuda'), torch.tensor([K - 1], device='cuda')])
    want = x[:, rows].double().t() @ dz
    # SiLU: dz of M rows is rounded before it is summed, z too (its slope changes by at most 0.5 a unit, z is below 1): even, M of them
    _check(dw[rows][:, columns], want, dtype, added=8 * HALF[dtype] / M ** 0.5 if act == 'silu' else 0.0)
    assert spmm_cpp.dense_status() == 0
    again, = torch.autograd.grad(spmm_cpp.linear(x, w, activation=act), w, dy)
    assert torch.equal(again, dw)


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('M,K,N,act', [(70_001, 24, 40, None), (66_000, 300, 520, None), (66_000, 72, 24_000, 'relu'), (70_003, 40, 24_008, None)])
def test_whole_numbers_of_many_rows_are_exact(M, K, N, act, dtype):
    """Sums below 2^24 of whole numbers: bit for bit, whatever chains and ranges they come in; bias gradients with them."""
    import spmm_cpp
    gen = torch.Generator(device='cuda').manual_seed(M + K)
    x = torch.randint(-2, 3, (M, K), device='cuda', generator=gen).to(dtype)
    w = torch.randint(-1, 2, (K, N), device='cuda', generator=gen).to(dtype).requires_grad_()
    b = torch.full((N,), 0.5, device='cuda', dtype=dtype, requires_grad=True)
    dy = torch.randint(-1, 2, (M, N), device='cuda', generator=gen, dtype=torch.int8).to(dtype)
    dw, db = torch.autograd.grad(spmm_cpp.linear(x, w, b, activation=act), [w, b], dy)
    columns = torch.tensor([0, 3, N // 2, N - 8, N - 1], device='cuda')
    z = x.double() @ w.detach()[:, columns].double() + 0.5
    dz = dy[:, columns].double() * ((z > 0) if act else 1)
    assert torch.equal(dw[:, columns], (x.double().t() @ dz).to(dtype)) and torch.equal(db[columns], dz.sum(0).to(dtype))
    assert spmm_cpp.dense_status() == 0


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('M,K,N', [(300, 33, 40), (511, 301, 530), (100, 1, 300), (600, 99, 19_306), (1_000, 70, 19_201)])
@pytest.mark.parametrize('act', [None, 'relu'])
def test_gradients_of_one_range_and_odd_widths(M, K, N, act, dtype):
    """Few rows, or so many panels that each has all rows: accumulators go to the result directly, where lanes of a warp have rows and others have none."""
    import spmm_cpp
    gen = torch.Generator(device='cuda').manual_seed(M + K)
    x = torch.randint(-2, 3, (M, K), device='cuda', generator=gen).to(dtype)
    w = torch.randint(-1, 2, (K, N), device='cuda', generator=gen).to(dtype)
    dy = torch.randint(-1, 2, (M, N), device='cuda', generator=gen).to(dtype)
    for weight in (w.clone(), w.t().contiguous().t()):
        weight.requires_grad_()
        b = torch.full((N,), 0.5, device='cuda', dtype=dtype, requires_grad=True)
        dw, db = torch.autograd.grad(spmm_cpp.linear(x, weight, b, activation=act), [weight, b], dy)
        dz = dy.double() * ((x.double() @ w.double() + 0.5 > 0) if act else 1)
        assert torch.equal(dw, (x.double().t() @ dz).to(dtype)) and torch.equal(db, dz.sum(0).to(dtype))
    assert spmm_cpp.dense_status() == 0


@pytest.mark.parametrize('M,K,N', [(2000, 257, 128), (2000, 602, 128), (300, 1024, 41), (5000, 4096, 200), (40, 4097, 96), (700, 16_384, 130), (20_000, 300, 64)])
@pytest.mark.parametrize('signs', ['one', 'both'])
def test_products_of_many_columns_fp32(M, K, N, signs):
    """Three TF32 passes: chains of at most 1,024 columns whatever K is, forward and in x's gradient.  Of the sum of magnitudes S each element is off by the chain's share,
    2^-20.8 for the terms that the passes leave out and for the weight's tails, and the additions of K / 1,024 chains in fp32.  On average an accumulation is off by a step of
    the running sum at most: over a chain of n, n / 2 steps of a sum that grows evenly, and two thirds of n of one that grows with the square root, as those of both signs do."""
    import spmm_cpp
    gen = torch.Generator(device='cuda').manual_seed(K)
    make = torch.rand if signs == 'one' else torch.randn
    x, w = (make(s, device='cuda', generator=gen) for s in ((M, K), (K, N)))
    chains = 2.0 ** -24 * ((K + 1023) // 1024) + 2.0 ** -20.8
    want, size = x.double() @ w.double(), x.double().abs() @ w.double().abs()
    back = (torch.rand if signs == 'one' else torch.randn)(M, K, device='cuda', generator=gen)
    v = w.t().contiguous().requires_grad_(False)                   # [N x K]: x's gradient of a layer N -> K sums over K columns
    a = torch.zeros(M, N, device='cuda', requires_grad=True)
    dx, = torch.autograd.grad(spmm_cpp.linear(a, v), a, back)
    for got, exact, total in ((spmm_cpp.linear(x, w), want, size), (dx, back.double() @ v.double().t(), back.double().abs() @ v.double().abs().t())):
        assert float(((got.double() - exact).abs() / total).max()) <= CHAIN[torch.float32] * 2 + chains
        assert float((got.double() - exact).norm() / exact.norm()) <= 128 * 2.0 ** -23 * (1 / 2 if signs == 'one' else 2 / 3) + chains
    assert spmm_cpp.dense_status() == 0


@pytest.mark.parametrize('M,K,N', [(600, 1100, 257), (2001, 1030, 47), (150, 1600, 1600), (17, 1025, 1), (260, 4097, 128), (3000, 1040, 130), (40_000, 2100, 300)])
@pytest.mark.parametrize('act', [None, 'relu', 'gelu', 'silu'])
def test_whole_numbers_of_many_columns_are_exact_fp32(M, K, N, act):
    """Several chains with every epilogue: bias, activation, residual, what is kept for the gradient, panels and rows that end inside a tile.  Whole numbers: bit for bit
    but for GELU and SiLU, which see the exact z (an even number, so that there are none between -2 and 2 but 0)."""
    import spmm_cpp
    gen = torch.Generator(device='cuda').manual_seed(M + K + N)
    x, w, r, dy = (torch.randint(-1, 2, s, device='cuda', generator=gen).float() for s in ((M, K), (K, N), (M, N), (M, N)))
    x *= 2
    b = torch.ones(N, device='cuda') * 2
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    y = spmm_cpp.linear(x, w, b, residual=r, activation=act)
    z = x.detach().double() @ w.detach().double() + 2
    if act in ('gelu', 'silu'):
        value = z * (torch.sigmoid(z) if act == 'silu' else 0.5 * torch.erfc(-z * 0.5 ** 0.5))
        assert float((y.detach().double() - value - r.detach().double()).abs().max()) <= 2.0 ** -21 * float(z.abs().max())
        assert all(bool(torch.isfinite(g).all()) for g in torch.autograd.grad(y, leaves, dy))
    else:
        value, slope = (z.clamp(min=0), z > 0) if act else (z, torch.ones_like(z))
        assert torch.equal(y.detach(), (value + r.detach().double()).float())
        dz = dy.double() * slope
        for got, exact in zip(torch.autograd.grad(y, leaves, dy), (dz @ w.detach().double().t(), x.detach().double().t() @ dz, dz.sum(0), dy.double())):
            assert torch.equal(got, exact.float())
    assert spmm_cpp.dense_status() == 0


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('M,K,N', [(600, 65_536, 200), (300, 100_001, 40), (40, 40_000, 300), (700, 8_200, 64), (20_000, 16_400, 136)])
def test_products_of_many_columns(M, K, N, dtype):
    """Chains of K's columns in the product and in x's gradient, whose sum runs over the outputs."""
    import spmm_cpp
    gen = torch.Generator(device='cuda').manual_seed(K)
    x, w = _positive(gen, M, K, dtype=dtype), _positive(gen, K, N, dtype=dtype) * (64 / K)
    rows = torch.arange(0, M, max(1, M // 300), device='cuda')
    y = spmm_cpp.linear(x, w)
    _check(y[rows], x[rows].double() @ w.double(), dtype)
    v = w.t().contiguous()                                         # [N x K]
    a = torch.zeros(M, N, device='cuda', dtype=dtype, requires_grad=True)
    dx, = torch.autograd.grad(spmm_cpp.linear(a, v), a, x)
    _check(dx[rows], x[rows].double() @ v.double().t(), dtype)
    assert spmm_cpp.dense_status() == 0


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('M,K,N,act', [(600, 33_000, 257, 'relu'), (3001, 66_000, 47, None), (40, 40_000, 520, 'relu'), (20_000, 33_001, 130, 'relu'), (33, 70_000, 5, 'relu')])
def test_whole_numbers_of_many_columns_are_exact(M, K, N, act, dtype):
    """Several chains with bias, residual and ReLU's bits, panels and rows that end inside a tile: bit for bit."""
    import spmm_cpp
    gen = torch.Generator(device='cuda').manual_seed(K + N)
    x, w = (torch.randint(-1, 2, s, device='cuda', generator=gen, dtype=torch.int8).to(dtype) for s in ((M, K), (K, N)))
    r = torch.randint(-2, 3, (M, N), device='cuda', generator=gen).to(dtype)
    b = torch.full((N,), 0.5, device='cuda', dtype=dtype, requires_grad=True)
    dy = torch.randint(-1, 2, (M, N), device='cuda', generator=gen).to(dtype)
    y = spmm_cpp.linear(x, w, b, residual=r, activation=act)
    z = (x.float() @ w.float()).double() + 0.5                     # whole numbers below 2^24: exact in fp32
    assert torch.equal(y.detach(), ((z.clamp(min=0) if act else z) + r.double()).to(dtype))
    db, = torch.autograd.grad(y, b, dy)
    assert torch.equal(db, (dy.double() * ((z > 0) if act else 1)).sum(0).to(dtype))
    assert spmm_cpp.dense_status() == 0


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('M,K,N', [(16, 1 << 20, 48), (32, 1_500_001, 40), (1, 1 << 21, 64), (5, 600_006, 33)])
@pytest.mark.parametrize('transposed', [False, True])
def test_products_of_few_rows_and_many_columns(M, K, N, transposed, dtype):
    """Every warp's chains of a share of K, with whole and with odd alignments."""
    import spmm_cpp
    gen = torch.Generator(device='cuda').manual_seed(K + M)
    x, w = _positive(gen, M, K, dtype=dtype), _positive(gen, K, N, dtype=dtype) * (64 / K)
    w = w.t().contiguous().t() if transposed else w
    _check(spmm_cpp.linear(x, w), x.double() @ w.double(), dtype)


@pytest.mark.parametrize('dtype,M,K,N', [(torch.float32, 600, 2100, 1200), (torch.float16, 600, 20_000, 9_000), (torch.bfloat16, 70_000, 72, 300)])
def test_chains_captured_and_on_two_streams(dtype, M, K, N):
    """Layers whose products, x's gradients or weight gradients take several chains, two at once and replayed with other inputs: the eager numbers, bit for bit."""
    import spmm_cpp
    gen = torch.Generator(device='cuda').manual_seed(N)
    x, w, dy = _positive(gen, M, K, dtype=dtype), _positive(gen, K, N, dtype=dtype) * (4 / K), _positive(gen, M, N, dtype=dtype) * (4 / N)

    def both(a, b):
        y = spmm_cpp.linear(a, b, activation='silu')
        return (y.detach(), *torch.autograd.grad(y, [a, b], dy))

    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    want = both(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            there = both(a, b)
        here = both(a, b)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(want, there)) and all(torch.equal(p, q) for p, q in zip(want, here))
    torch.cuda.synchronize()
    del want, there, here
    c, d = x.clone().requires_grad_(), w.clone().requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both(c, d)
    with torch.no_grad():
        c.copy_(_positive(gen, M, K, dtype=dtype))
    graph.replay()
    torch.cuda.synchronize()
    e, f = c.detach().clone().requires_grad_(), d.detach().clone().requires_grad_()
    assert all(torch.equal(p, q) for p, q in zip(got, both(e, f)))
    assert spmm_cpp.dense_status() == 0
