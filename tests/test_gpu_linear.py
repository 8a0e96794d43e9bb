"""spmm_cpp.linear - activation(x w + b) + r in one kernel, and its gradients - against float64.  Needs a GPU.

Tolerances.  S = |x| |w| is the sum of the magnitudes that go into an element.  A product's sum in fp32 accumulators that truncate is off by at most one
step (2^-23) of the running sum for every accumulation, K / 8 of them and fewer, and the fp32 product drops three terms of 2^-22: SUM(K) = (K / 8 + 16) *
2^-23 * 3 of S.  The result adds half a step of its type.  Behind an activation the slope is at most 1.13.  The gradient rounds z (its slope changes by at
most 0.8 a unit) and dz to the type before it is multiplied: HALF * (|dz| + 0.8 |z| |dy|) for each, which goes through |w| or |x| like dz itself.
Inputs that are small whole numbers make all of this exact: then the result is the rounded number itself."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SHAPES = [(1, 1, 1), (1, 256, 256), (2, 7, 5), (16, 1024, 1024), (17, 64, 64), (31, 100, 47), (32, 33, 130), (33, 8, 8), (100, 602, 41), (127, 256, 16), (128, 128, 48),
          (129, 100, 256), (255, 48, 300), (256, 256, 256), (257, 300, 512), (1000, 16, 1024), (1500, 1024, 65), (20001, 256, 256), (40000, 64, 10), (38000, 72, 200),
          (5, 32, 32), (127, 7, 11), (129, 1, 3), (3000, 32, 16), (9999, 31, 29), (150000, 7, 11), (4096, 4, 4)]


def _acts64(name, z):
    """(value, slope)"""
    if name == 'relu':
        return z.clamp(min=0), (z > 0).double()
    if name == 'gelu':
        cdf = 0.5 * torch.erfc(-z * math.sqrt(0.5))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == 'silu':
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    return z, torch.ones_like(z)


def _whole(gen, *shape, most=2):
    return torch.randint(-most, most + 1, shape, device='cuda', generator=gen).float()


def _grads(y, dy, *tensors):
    return torch.autograd.grad(y, [t for t in tensors if t is not None], dy)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('M,K,N', SHAPES)
@pytest.mark.parametrize('act', [None, 'relu'])
def test_whole_numbers_are_exact(dtype, M, K, N, act):
    import spmm_cpp
    gen = torch.Generator(device='cuda').manual_seed(M + 3 * K + 7 * N)
    out_in = (M + K) % 2 == 1
    x = _whole(gen, M, K).to(dtype).requires_grad_()
    w = _whole(gen, N, K, most=1).to(dtype).t() if out_in else _whole(gen, K, N, most=1).to(dtype)
    w = w.detach().requires_grad_()
    b = (_whole(gen, N) + 0.5).to(dtype).requires_grad_()          # no z is zero
    r = _whole(gen, M, N).to(dtype).requires_grad_()
    dy = _whole(gen, M, N, most=1).to(dtype)
    y = spmm_cpp.linear(x, w, b, residual=r, activation=act)
    z = x.detach().double() @ w.detach().double() + b.detach().double()
    value, slope = _acts64(act, z)
    assert y.dtype == dtype and y.shape == (M, N)
    assert torch.equal(y.detach(), (value + r.detach().double()).to(dtype))
    dx, dw, db, dr = _grads(y, dy, x, w, b, r)
    dz = dy.double() * slope
    assert torch.equal(dx, (dz @ w.detach().double().t()).to(dtype))
    assert torch.equal(dw, (x.detach().double().t() @ dz).to(dtype)) and dw.shape == w.shape
    assert torch.equal(db, dz.sum(0).to(dtype)) and torch.equal(dr, dy)
    with torch.no_grad():
        assert torch.equal(spmm_cpp.linear(x, w, b, residual=r, activation=act), y)
        assert torch.equal(spmm_cpp.linear(x, w, activation=act), _acts64(act, z - b.double())[0].to(dtype))
    assert spmm_cpp.dense_status() == 0


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('M,K,N', SHAPES)
@pytest.mark.parametrize('act', ['gelu', 'silu'])
def test_smooth_activations_match_float64(dtype, M, K, N, act):
    import spmm_cpp
    gen = torch.Generator(device='cuda').manual_seed(M + 5 * K + 11 * N)
    x = torch.randn(M, K, device='cuda', generator=gen).to(dtype).requires_grad_()
    w = (torch.randn(K, N, device='cuda', generator=gen) / K ** 0.5).to(dtype).requires_grad_()
    b = torch.randn(N, device='cuda', generator=gen).to(dtype).requires_grad_()
    r = torch.randn(M, N, device='cuda', generator=gen).to(dtype).requires_grad_()
    dy = torch.randn(M, N, device='cuda', generator=gen).to(dtype)
    y = spmm_cpp.linear(x, w, b, residual=r, activation=act)
    got = _grads(y, dy, x, w, b, r)
    xd, wd, bd, rd, dyd = (t.detach().double() for t in (x, w, b, r, dy))
    half, sums = HALF[dtype], lambda n: (n / 8 + 16) * 3 * 2.0 ** -23
    z = xd @ wd + bd
    value, slope = _acts64(act, z)
    ez = sums(K) * (xd.abs() @ wd.abs() + bd.abs())
    want = value + rd
    small = 2.0 ** -22 * (1 + z.abs())                             # of the activation itself, and of the residual's addition
    subnormal = 2.0 ** -25 if dtype == torch.float16 else 0.0
    assert bool(((y.detach().double() - want).abs() <= half * want.abs() + 1.14 * ez + small * (1 + rd.abs()) + subnormal).all())
    dz = dyd * slope
    edz = half * (dz.abs() + 0.81 * z.abs() * dyd.abs()) * 1.01 + (ez + 2 * small) * dyd.abs() + subnormal
    for name, grad, exact, error, terms, count in (('dx', got[0], dz @ wd.t(), edz @ wd.abs().t(), dz.abs() @ wd.abs().t(), N),
                                                   ('dw', got[1], xd.t() @ dz, xd.abs().t() @ edz, xd.abs().t() @ dz.abs(), min(M, 32768)),
                                                   ('db', got[2], dz.sum(0), edz.sum(0), dz.abs().sum(0), min(M, 512))):
        bound = half * exact.abs() + error * 1.01 + sums(count) * terms + subnormal
        worst = ((grad.double() - exact).abs() / bound.clamp(min=1e-300)).max()
        assert float(worst) <= 1, f'{name}: {float(worst):.2f} of the bound'
    assert torch.equal(got[3], dy)
    again = spmm_cpp.linear(x, w, b, residual=r, activation=act)
    assert torch.equal(again, y) and all(torch.equal(p, q) for p, q in zip(_grads(again, dy, x, w, b, r), got))
    assert spmm_cpp.dense_status() == 0


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('M', [5, 700])
def test_strides_offsets_and_broadcasts(dtype, M):
    """Operands that are slices, transposes and expansions, every gradient against that of contiguous copies."""
    import spmm_cpp
    gen = torch.Generator(device='cuda').manual_seed(M)
    K, N = 40, 24

    def wide(rows, cols, kind):
        if kind == 'slice':
            return _whole(gen, rows, cols + 5).to(dtype)[:, 3:3 + cols]
        if kind == 'transpose':
            return _whole(gen, cols, rows).to(dtype).t()
        if kind == 'rows':
            return _whole(gen, 2 * rows, cols).to(dtype)[::2]
        if kind == 'padded':
            return _whole(gen, rows, cols + 8).to(dtype)[:, :cols]
        return _whole(gen, 1, cols).to(dtype).expand(rows, cols)

    for kx, kw, kr, kd in (('slice', 'slice', 'slice', 'slice'), ('transpose', 'transpose', 'transpose', 'transpose'), ('rows', 'rows', 'rows', 'rows'),
                           ('padded', 'padded', 'padded', 'padded'), ('one', 'one', 'one', 'one')):
        x, w, r, dy = wide(M, K, kx), wide(K, N, kw), wide(M, N, kr), wide(M, N, kd)
        b = _whole(gen, 2 * N).to(dtype)[::2] + 0.5
        views = [t.detach().requires_grad_() for t in (x, w, b, r)]
        plain = [t.detach().clone(memory_format=torch.contiguous_format).requires_grad_() for t in (x, w, b, r)]
        a = spmm_cpp.linear(views[0], views[1], views[2], residual=views[3], activation='relu')
        c = spmm_cpp.linear(plain[0], plain[1], plain[2], residual=plain[3], activation='relu')
        assert torch.equal(a, c), (kx, kw)
        for p, q in zip(_grads(a, dy, *views), _grads(c, dy.contiguous(), *plain)):
            assert torch.equal(p, q), (kx, kw)
        wanted = (x.double() @ w.double() + b.double()).clamp(min=0) + r.double()
        assert torch.equal(c.detach(), wanted.to(dtype))
    # a broadcast input's gradient is summed by autograd
    row = torch.ones(1, K, device='cuda', dtype=dtype, requires_grad=True)
    w = _whole(gen, K, N).to(dtype)
    spmm_cpp.linear(row.expand(M, K), w).sum().backward()
    assert torch.equal(row.grad, (w.double().sum(1) * M).to(dtype)[None]) or dtype != torch.float32


def test_only_what_is_asked_for():
    import spmm_cpp
    x, w, b, r = (torch.randn(s, device='cuda') for s in ((300, 20), (20, 30), (30,), (300, 30)))
    for asked in range(1, 16):
        tensors = [t.clone().requires_grad_(bool(asked >> i & 1)) for i, t in enumerate((x, w, b, r))]
        y = spmm_cpp.linear(tensors[0], tensors[1], tensors[2], residual=tensors[3], activation='gelu')
        y.backward(torch.ones_like(y))
        for i, t in enumerate(tensors):
            assert (t.grad is not None) == bool(asked >> i & 1)
    assert not spmm_cpp.linear(x, w).requires_grad


@pytest.mark.parametrize('M,K,N', [(40, 24, 16), (5000, 24, 16), (1000, 9, 32), (700, 256, 264), (700, 300, 40), (20000, 64, 96), (900, 40, 41)])
@pytest.mark.parametrize('act', [None, 'relu', 'gelu', 'silu'])
def test_every_subset_of_gradients_is_the_same(M, K, N, act):
    """Which gradients are asked for decides which kernels run (dz on the way to the weight gradient, by itself, kept or not): the numbers are those of all of them, but
    for sums that a kernel of its own takes in another order."""
    import spmm_cpp
    gen = torch.Generator(device='cuda').manual_seed(M + N)
    base = [torch.randn(*s, device='cuda', generator=gen).bfloat16() for s in ((M, K), (K, N), (N,), (M, N))]
    dy = torch.randn(M, N, device='cuda', generator=gen).bfloat16()
    all_leaves = [t.clone().requires_grad_() for t in base]
    want = _grads(spmm_cpp.linear(*all_leaves[:3], residual=all_leaves[3], activation=act), dy, *all_leaves)
    for asked in range(1, 16):
        leaves = [t.clone().requires_grad_(bool(asked >> i & 1)) for i, t in enumerate(base)]
        y = spmm_cpp.linear(*leaves[:3], residual=leaves[3], activation=act)
        got = iter(_grads(y, dy, *[t for t in leaves if t.requires_grad]))
        for i in range(4):
            if asked >> i & 1:
                g = next(got)
                if i == 2:                                         # one step of the result, and the order of M sums
                    assert float((g.double() - want[i].double()).abs().max()) <= (2.0 ** -7 + M * 2.0 ** -24) * float(want[i].abs().max())
                else:
                    assert torch.equal(g, want[i]), (asked, i)
    assert spmm_cpp.dense_status() == 0


def test_gradients_against_differences():
    """Central differences of f = sum(c y) along random directions in fp32: truncation h^2 / 6 of third derivatives (at most 2 a unit of z) and the
    rounding of y, 2^-22 (|y| + S) / 2h for each, added as if they were independent, eight deviations."""
    import spmm_cpp
    gen = torch.Generator(device='cuda').manual_seed(2)
    M, K, N, h = 200, 32, 24, 2.0 ** -6
    base = [torch.randn(M, K, device='cuda', generator=gen), torch.randn(K, N, device='cuda', generator=gen) / K ** 0.5, torch.randn(N, device='cuda', generator=gen),
            torch.randn(M, N, device='cuda', generator=gen)]
    c = torch.randn(M, N, device='cuda', generator=gen)
    for act in ('gelu', 'silu'):
        leaves = [t.clone().requires_grad_() for t in base]
        y = spmm_cpp.linear(leaves[0], leaves[1], leaves[2], residual=leaves[3], activation=act)
        grads = _grads(y, c, *leaves)
        for i, t in enumerate(base):
            v = torch.randn(t.shape, device='cuda', generator=gen)
            v /= max(1.0, float(v.norm()) / math.sqrt(M))           # a change of z of order one
            f = []
            for sign in (1, -1):
                moved = [u + sign * h * v if j == i else u for j, u in enumerate(base)]
                f.append(float((spmm_cpp.linear(moved[0], moved[1], moved[2], residual=moved[3], activation=act).double() * c.double()).sum()))
            slope = (f[0] - f[1]) / (2 * h)
            want = float((grads[i].double() * v.double()).sum())
            moved_z = (v @ base[1] if i == 0 else base[0] @ v if i == 1 else v.expand(M, N)).double().abs() if i < 3 else torch.zeros(M, N, device='cuda', dtype=torch.float64)
            truncation = float((c.abs().double() * 2 * moved_z ** 3).sum()) * h * h / 6
            rounding = 8 * float((c.abs() * (y.detach().abs() + 4) * 2.0 ** -22).norm()) / (2 * h)
            assert abs(slope - want) <= truncation + rounding, (act, i, slope, want)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('M', [8, 500])
def test_what_is_not_finite_stays_in_its_row(dtype, M):
    import spmm_cpp
    for act in (None, 'relu', 'gelu', 'silu'):
        x, w = torch.ones(M, 64, device='cuda', dtype=dtype), torch.full((64, 40), 0.125, device='cuda', dtype=dtype)
        x[3, 5], x[6, 7] = float('nan'), float('inf')
        y = spmm_cpp.linear(x, w, activation=act)
        assert bool(torch.isnan(y[3]).all()) and not bool(torch.isfinite(y[6]).any())
        rest = [i for i in range(M) if i not in (3, 6)]
        assert bool(torch.isfinite(y[rest]).all())


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('M,K,N', [(100_000, 5, 6), (100_000, 30, 7), (100_000, 3, 32), (3000, 64, 40), (20, 64, 40)])
def test_gradients_that_are_not_finite_stay_in_their_rows(dtype, M, K, N):
    """A NaN or an infinity in a row of the incoming gradient reaches that row of x's gradient, and no other, whichever rows share its place in a tile."""
    import spmm_cpp
    for act in (None, 'relu', 'gelu'):
        x = torch.ones(M, K, device='cuda', dtype=dtype, requires_grad=True)
        w = torch.full((K, N), 0.125, device='cuda', dtype=dtype)
        dy = torch.ones(M, N, device='cuda', dtype=dtype)
        dy[3, N - 1], dy[7, 0], dy[M - 5, 0] = float('nan'), float('inf'), float('nan')
        dx, = torch.autograd.grad(spmm_cpp.linear(x, w, activation=act), x, dy)
        bad = sorted(set((~torch.isfinite(dx)).any(1).nonzero().view(-1).tolist()))
        assert bad == sorted({3, 7, M - 5}), (act, bad[:10])


def test_rows_behind_the_result_are_left_alone():
    """The padded rows' columns aside, nothing but the result is written: results of many shapes in one buffer's neighbourhood."""
    import ctypes
    import spmm_cpp
    L = spmm_cpp.lib()

    class Args(ctypes.Structure):
        _fields_ = [(n, ctypes.c_void_p) for n in ('x', 'w', 'head', 'tail', 'bias', 'residual', 'y', 'z', 'bits')] + \
                   [(n, ctypes.c_int64) for n in ('ldx', 'ldw', 'ldb', 'ldr', 'ldy', 'ldz', 'ldbits', 'M')] + \
                   [(n, ctypes.c_int32) for n in ('N', 'K', 'type', 'act', 'out_in', 'pad')]

    for M, K, N in ((5, 16, 40), (300, 16, 24), (300, 64, 40), (129, 8, 200), (1, 8, 8), (511, 128, 264)):
        x, w = torch.ones(M, K, device='cuda', dtype=torch.bfloat16), torch.ones(K, N, device='cuda', dtype=torch.bfloat16)
        y = torch.full((M + 2, N + 8), 7.0, device='cuda', dtype=torch.bfloat16)
        z = y.clone()
        a = Args(x=x.data_ptr(), w=w.data_ptr(), y=y[1:].data_ptr(), z=z[1:].data_ptr(), ldx=K, ldw=N, ldy=N + 8, ldz=N + 8, M=M, N=N, K=K, type=1, act=2)
        assert L.dg_linear(ctypes.byref(a), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
        torch.cuda.synchronize()
        assert bool((z[1:-1, :N] == K).all())
        for t in (y, z):
            assert bool((t[0] == 7).all()) and bool((t[-1] == 7).all()) and bool((t[:, N:] == 7).all())


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_captured_and_on_two_streams(dtype):
    import spmm_cpp
    gen = torch.Generator(device='cuda').manual_seed(1)
    x, w, b, r, dy = (_whole(gen, *s).to(dtype) for s in ((900, 64), (64, 72), (72,), (900, 72), (900, 72)))
    leaves = [t.clone().requires_grad_() for t in (x, w, b, r)]

    def both(ts):
        y = spmm_cpp.linear(ts[0], ts[1], ts[2], residual=ts[3], activation='silu')
        return (y.detach(), *_grads(y, dy, *ts))

    want = both(leaves)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):                                             # the same weight on two streams at once
        with torch.cuda.stream(side):
            there = both(leaves)
        here = both(leaves)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(want, there)) and all(torch.equal(p, q) for p, q in zip(want, here))
    torch.cuda.synchronize()
    fresh = [t.detach().clone().requires_grad_() for t in leaves]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both(fresh)
    with torch.no_grad():
        fresh[0].copy_(_whole(gen, 900, 64))
    graph.replay()
    torch.cuda.synchronize()
    eager = [t.detach().clone().requires_grad_() for t in fresh]
    assert all(torch.equal(p, q) for p, q in zip(got, both(eager)))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_first_call_of_a_thread(dtype):
    """A thread whose first use of the device is one of these calls, memory for them lying ready."""
    import threading
    import spmm_cpp
    x, w, dy = torch.ones(300, 64, device='cuda', dtype=dtype), torch.ones(64, 40, device='cuda', dtype=dtype, requires_grad=True), torch.ones(300, 40, device='cuda', dtype=dtype)
    want = spmm_cpp.linear(x, w)
    del want
    out = []

    def call():
        try:
            out.append(spmm_cpp.linear(x, w).detach().float().mean())
            out.append(spmm_cpp.dense_nt(x, w.detach(), transposed=True) if dtype == torch.float32 else out[0])
        except Exception as e:
            out.append(e)
    for _ in range(3):
        thread = threading.Thread(target=call)
        thread.start(), thread.join()
    assert not [v for v in out if isinstance(v, Exception)], out
    assert all(float(v.mean()) == 64 for v in out)
    y = spmm_cpp.linear(x, w)
    assert float(torch.autograd.grad(y, w, dy)[0].float().mean()) == 300


def test_padding_of_fp32_rows_is_zero():
    """Products read padded rows of fp32 operands whole; results and x's gradients of odd widths have zeros there, whatever the memory held."""
    import spmm_cpp
    junk = torch.full((64, 1 << 16), float('nan'), device='cuda')
    del junk
    for M in (40, 5000):
        x, w = torch.ones(M, 33, device='cuda', requires_grad=True), torch.ones(33, 41, device='cuda')
        y = spmm_cpp.linear(x, w, activation='gelu')
        dx, = torch.autograd.grad(y, x, torch.ones_like(y))
        for t, cols, width in ((y.detach(), 41, 44), (dx, 33, 36)):
            assert t.stride(0) == width and bool((t.as_strided((M, width - cols), (width, 1), cols) == 0).all())


def test_refusals():
    import spmm_cpp
    x, w = torch.ones(4, 6, device='cuda'), torch.ones(6, 5, device='cuda')
    for args, kw in (((x, w.t()), {}), ((x.cpu(), w), {}), ((x, w.cpu()), {}), ((x, w.bfloat16()), {}), ((x.double(), w.double()), {}), ((x[0], w), {}),
                     ((x, w, torch.ones(6, device='cuda')), {}), ((x, w, torch.ones(5)), {}), ((x, w), dict(residual=torch.ones(1, 5, device='cuda'))),
                     ((x, w), dict(residual=torch.ones(4, 5, device='cuda').half())), ((x[:, :0], w[:0]), {}), ((x, w[:, :0]), {})):
        with pytest.raises(RuntimeError, match='linear'):
            spmm_cpp.linear(*args, **kw)
    with pytest.raises(ValueError):
        spmm_cpp.linear(x, w, activation='tanh')
    y = spmm_cpp.linear(x[:0], w.requires_grad_())
    assert y.shape == (0, 5)
    y.sum().backward()
    assert bool((w.grad == 0).all())
    y = spmm_cpp.linear(x, w, activation='gelu')
    with torch.no_grad():
        w.add_(1)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()
    y = spmm_cpp.linear(x, w, activation='gelu')
    with pytest.raises(RuntimeError, match='differentiated again'):
        torch.autograd.grad(y.sum(), w, create_graph=True)
    y.sum().backward()
    with pytest.raises(RuntimeError, match='second time'):
        y.sum().backward()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('M,K,N', [(4804, 34, 539), (3000, 40, 298), (20000, 33, 130), (700, 64, 1100), (300, 48, 65), (40000, 36, 257), (5000, 40, 97)])
def test_relu_gradients_of_wide_layers_are_exact(M, K, N, dtype):
    """Results in several panels, the last one with pieces beyond the matrix: what ReLU keeps is every row's own.  Small whole numbers: sums stay below
    2^24, so that results are the exact ones, rounded once."""
    import spmm_cpp
    g = torch.Generator(device='cuda').manual_seed(M + N)
    x, w, b, dy = (torch.randint(-2, 3, size, device='cuda', generator=g).to(dtype) for size in ((M, K), (K, N), (N,), (M, N)))
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = spmm_cpp.linear(x, w, b, activation='relu')
    grads = torch.autograd.grad(y, leaves, dy)
    z = x.detach().double() @ w.detach().double() + b.detach().double()
    dz = dy.double() * (z > 0)
    for got, want in zip((y, *grads), (z.clamp(min=0), dz @ w.detach().double().t(), x.detach().double().t() @ dz, dz.sum(0))):
        assert torch.equal(got.detach(), want.float().to(dtype))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('M,K,N', [(459, 1, 46), (9, 1, 78), (1, 1, 215), (684, 1, 327), (459, 46, 1), (3, 272, 1), (20, 33, 1)])
def test_one_input_or_output_with_strides(M, K, N, dtype):
    """A weight of one row or column, whose stride along it says nothing: every second element of a wider one, and its transpose.  Whole numbers, as above."""
    import spmm_cpp
    g = torch.Generator(device='cuda').manual_seed(M + N)
    x, dy = (torch.randint(-2, 3, size, device='cuda', generator=g).to(dtype) for size in ((M, K), (M, N)))
    wide = torch.randint(-2, 3, (2 * K, 2 * N), device='cuda', generator=g).to(dtype)
    for w in (wide[:K, ::2], wide[::2, :N], wide[:K, :N].t().contiguous().t(), wide[:K, :N].contiguous()):
        leaves = [x.detach().requires_grad_(), w.detach().requires_grad_()]
        y = spmm_cpp.linear(*leaves)
        grads = torch.autograd.grad(y, leaves, dy)
        for got, want in zip((y, *grads), (x.double() @ w.double(), dy.double() @ w.double().t(), x.double().t() @ dy.double())):
            assert torch.equal(got.detach(), want.float().to(dtype))
