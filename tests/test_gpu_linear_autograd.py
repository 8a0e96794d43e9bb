"""spmm_cpp.linear as a node of autograd: what it keeps between the passes, and calls that it has to refuse.  Needs a GPU."""
import pytest
import torch

pytestmark = pytest.mark.gpu
CASES = [(700, 256, 264, torch.float32), (700, 40, 41, torch.float32), (700, 256, 264, torch.bfloat16), (5000, 41, 33, torch.float16), (700, 300, 40, torch.bfloat16),
         (9, 40, 48, torch.bfloat16), (9, 40, 48, torch.float32), (300, 7, 11, torch.float32)]


def _leaves(M, K, N, dtype, seed=1):
    g = torch.Generator(device='cuda').manual_seed(seed)
    shapes = ((M, K), (K, N), (N,), (M, N))
    return [torch.randint(-2, 3, s, device='cuda', generator=g).to(dtype).requires_grad_() for s in shapes], torch.randint(-2, 3, (M, N), device='cuda', generator=g).to(dtype)


@pytest.mark.parametrize('M,K,N,dtype', CASES)
@pytest.mark.parametrize('act', [None, 'relu', 'gelu'])
@pytest.mark.parametrize('transposed', [False, True])
def test_saved_tensor_hooks_have_everything(M, K, N, dtype, act, transposed):
    """Offloaded to the host and brought back, in other memory and with other strides: the same gradients; a bias's may be summed in another order (one step)."""
    import spmm_cpp
    leaves, dy = _leaves(M, K, N, dtype)
    if transposed:
        leaves[1] = leaves[1].detach().t().contiguous().t().requires_grad_()
    want = torch.autograd.grad(spmm_cpp.linear(leaves[0], leaves[1], leaves[2], residual=leaves[3], activation=act), leaves, dy)
    packed = []

    def pack(t):
        packed.append(t.numel() * t.element_size())
        return t.cpu()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.cuda()):
        y = spmm_cpp.linear(leaves[0], leaves[1], leaves[2], residual=leaves[3], activation=act)
    assert len(packed) >= 2 and sum(packed) >= (M * K + K * N) * dtype.itemsize
    got = torch.autograd.grad(y, leaves, dy)
    for i, (p, q) in enumerate(zip(got, want)):
        if i == 2 and act == 'gelu':
            assert float((p.double() - q.double()).abs().max()) <= (2.0 ** -7 + M * 2.0 ** -24) * float(q.abs().max())
        else:
            assert torch.equal(p, q), i


def test_offloaded_memory_is_free():
    """Between the passes nothing of x, z or their copies stays on the device: what is held is the result."""
    import spmm_cpp
    a, w = torch.randn(60_000, 258, device='cuda', dtype=torch.bfloat16, requires_grad=True), torch.randn(258, 256, device='cuda', dtype=torch.bfloat16, requires_grad=True)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
        y = spmm_cpp.linear(a * 2, w, activation='gelu')
    assert torch.cuda.memory_allocated() - before <= y.untyped_storage().nbytes() + (1 << 20)
    y.backward(torch.ones_like(y))
    assert a.grad.shape == a.shape and w.grad.shape == w.shape


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_checkpoints(dtype):
    import spmm_cpp
    from torch.utils.checkpoint import checkpoint
    leaves, dy = _leaves(600, 48, 56, dtype)

    def layer(x, w, b, r):
        return spmm_cpp.linear(spmm_cpp.linear(x, w, b, residual=r, activation='silu'), w.t(), activation='relu')

    up = torch.ones(600, 48, device='cuda', dtype=dtype)
    want = torch.autograd.grad(layer(*leaves), leaves, up)
    got = torch.autograd.grad(checkpoint(layer, *leaves, use_reentrant=False), leaves, up)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize('M,K,N,dtype', CASES)
def test_changes_in_place_of_what_is_not_needed(M, K, N, dtype):
    """A layer whose weight is frozen does not need x again; one that read a copy of x (odd rows) has the copy."""
    import spmm_cpp
    leaves, dy = _leaves(M, K, N, dtype)
    x, w = leaves[0], leaves[1].detach()
    want, = torch.autograd.grad(spmm_cpp.linear(x, w, activation='relu'), x, dy)
    h = x * 1
    y = spmm_cpp.linear(h, w, activation='relu')
    with torch.no_grad():
        h.add_(1)
    assert torch.equal(torch.autograd.grad(y, x, dy)[0], want)
    h, w = x.detach().clone(), leaves[1]
    y = spmm_cpp.linear(h, w, activation='relu')
    h.add_(1)
    if dtype != torch.float32 and K % 8 and N > 32:                  # 16-bit rows of no whole 16-byte pieces
        assert torch.equal(torch.autograd.grad(y, w, dy)[0], torch.autograd.grad(spmm_cpp.linear(x.detach(), w, activation='relu'), w, dy)[0])
    elif K % 4 == 0 or K <= 32 and N <= 32:
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            torch.autograd.grad(y, w, dy)


def test_graphs_that_are_kept_and_that_are_not():
    import spmm_cpp
    leaves, dy = _leaves(300, 40, 48, torch.bfloat16)
    y = spmm_cpp.linear(leaves[0], leaves[1], leaves[2], residual=leaves[3], activation='gelu')
    first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    second = torch.autograd.grad(y, leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(first, second))
    with pytest.raises(RuntimeError, match='second time'):
        torch.autograd.grad(y, leaves, dy)


def test_forward_mode_is_refused():
    """A tangent would be lost without a word."""
    import spmm_cpp
    import torch.autograd.forward_ad as fwd
    leaves, dy = _leaves(40, 40, 48, torch.float32)
    for i in range(4):
        with fwd.dual_level():
            args = [t.detach() for t in leaves]
            args[i] = fwd.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(RuntimeError, match='linear: tangents'):
                spmm_cpp.linear(args[0], args[1], args[2], residual=args[3])
    with fwd.dual_level():
        assert spmm_cpp.linear(*[t.detach() for t in leaves[:3]]).shape == (40, 48)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('M,K,N', [(5, 40, 24), (700, 40, 24), (700, 40, 41), (300, 7, 11)])
def test_broadcast_inputs(M, K, N, dtype):
    """A row for all of x, a number for all of a row of the residual: autograd sums the gradients.  Whole numbers below the type's exact ones in every row, and sums of them
    that fp32 holds: the rounded sum itself."""
    import spmm_cpp
    g = torch.Generator(device='cuda').manual_seed(M + N)
    row = torch.ones(1, K, device='cuda', dtype=dtype, requires_grad=True)
    side = torch.ones(M, 1, device='cuda', dtype=dtype, requires_grad=True)
    w = torch.randint(-2, 3, (K, N), device='cuda', generator=g).to(dtype)
    y = spmm_cpp.linear(row.expand(M, K), w, residual=side.expand(M, N))
    y.backward(torch.ones((), device='cuda', dtype=dtype).expand(M, N))
    assert torch.equal(row.grad, (w.double().sum(1) * M).to(dtype)[None])
    assert torch.equal(side.grad, torch.full((M, 1), float(N), device='cuda', dtype=torch.float64).to(dtype))


@pytest.mark.parametrize('dtype', [torch.float32, torch.float16])
@pytest.mark.parametrize('M,K,N', [(12, 40, 48), (5000, 24, 16), (700, 256, 264), (700, 300, 40), (900, 40, 41), (600, 1100, 33)])
@pytest.mark.parametrize('act', [None, 'relu', 'gelu', 'silu'])
def test_every_subset_of_gradients(M, K, N, act, dtype):
    """Which gradients are asked for decides which kernels run; the numbers are those of all of them, but for the bias's, which kernels sum in different orders: one step
    of the result and the order of M sums."""
    import spmm_cpp
    gen = torch.Generator(device='cuda').manual_seed(M + N)
    base = [torch.randn(*s, device='cuda', generator=gen).to(dtype) for s in ((M, K), (K, N), (N,), (M, N))]
    dy = torch.randn(M, N, device='cuda', generator=gen).to(dtype)

    def grads(asked):
        leaves = [t.clone().requires_grad_(bool(asked >> i & 1)) for i, t in enumerate(base)]
        y = spmm_cpp.linear(*leaves[:3], residual=leaves[3], activation=act)
        got = iter(torch.autograd.grad(y, [t for t in leaves if t.requires_grad], dy))
        return [next(got) if t.requires_grad else None for t in leaves]

    want = grads(15)
    for asked in range(1, 15):
        for i, (p, q) in enumerate(zip(grads(asked), want)):
            assert (p is not None) == bool(asked >> i & 1)
            if p is None:
                continue
            if i == 2:
                step = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -10}[dtype]
                assert float((p.double() - q.double()).abs().max()) <= (step + M * 2.0 ** -24) * float(q.abs().max())
            else:
                assert torch.equal(p, q), (asked, i)
    assert spmm_cpp.dense_status() == 0
