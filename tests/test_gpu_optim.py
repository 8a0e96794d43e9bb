"""spmm_cpp.AdamW (one launch over all tensors, states in 32 or 8 bits, clipping by the global norm) against the formula in float64.  Needs a GPU.

Tolerances.  32 bits, fp32 parameters: a step is about ten roundings of half a step (2^-24 relative) on numbers no larger than p itself, m
or v: 16 * 2^-24 of the largest magnitude involved.  bf16 / fp16 parameters add the rounding of p: half a step of the type.  8 bits:
m and r move to a neighbour, at most one step of e4m3, which is 2^-3 of the value or 2^-9 / 448 of the block's largest."""
import copy
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
HYPER = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.05)
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SIZES = [(1,), (7,), (8,), (255,), (256,), (257,), (2047,), (2048,), (2049,), (33, 47), (100, 256), (5, 1)]


def _params(sizes, dtype, seed, scale=1.0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    params = []
    for i, size in enumerate(sizes):
        p = torch.nn.Parameter(torch.randn(size, device='cuda', generator=g).to(dtype))
        p.grad = (torch.randn(size, device='cuda', generator=g) * scale * 10.0 ** -(i % 4)).to(dtype)
        params.append(p)
    return params, g


def _regrad(params, g, scale=1.0):
    for i, p in enumerate(params):
        p.grad = (torch.randn(p.shape, device='cuda', generator=g) * scale * 10.0 ** -(i % 4)).to(p.dtype)


def _coef(params, max_norm):
    norm = math.sqrt(sum(float(p.grad.double().square().sum()) for p in params if p.grad is not None))
    return norm, min(1.0, max_norm / (norm + 1e-6)) if max_norm else 1.0


def _step64(p, grad, m, v, t, coef, lr=HYPER['lr'], betas=HYPER['betas'], eps=HYPER['eps'], weight_decay=HYPER['weight_decay']):
    b1, b2 = betas
    g = grad.double() * coef
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = p * (1 - lr * weight_decay) - lr * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + eps)
    return p, m, v


def _values(state):
    """The means an 8-bit state stands for, in float64: (m, r)."""
    out = []
    for name in ('exp_avg', 'root'):
        codes, scale = state[name].float().double().view(-1), state[name + '_scale'].double()
        out.append((codes * scale.repeat_interleave(256)[:codes.numel()]).view(state[name].shape))
    return out


def _blocks_top(x):
    flat = torch.zeros(x.numel() + (-x.numel()) % 256, dtype=torch.float64, device=x.device)
    flat[:x.numel()] = x.abs().view(-1)
    return flat.view(-1, 256).amax(1).repeat_interleave(256)[:x.numel()].view(x.shape)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('max_norm', [None, 0.5, 1e6])
def test_32_bit_steps_match_float64(dtype, max_norm):
    import spmm_cpp
    params, g = _params(SIZES, dtype, 1)
    opt = spmm_cpp.AdamW(params, max_norm=max_norm, **HYPER)
    m = [torch.zeros(p.shape, dtype=torch.float64, device='cuda') for p in params]
    v = [x.clone() for x in m]
    for t in range(1, 6):
        norm, coef = _coef(params, max_norm)
        before = [p.detach().double() for p in params]
        grads = [p.grad.clone() for p in params]
        opt.step()
        if max_norm:
            assert abs(float(opt.grad_norm) - norm) <= 2 * HALF[torch.float32] * norm
        for i, p in enumerate(params):
            assert torch.equal(p.grad, grads[i])
            want, m[i], v[i] = _step64(before[i], grads[i], m[i], v[i], t, coef)
            state = opt.state[p]
            assert int(state['step']) == t
            ulp = 16 * HALF[torch.float32]
            for got, exact in ((state['exp_avg'], m[i]), (state['exp_avg_sq'], v[i])):
                assert float((got.double() - exact).abs().max()) <= t * ulp * float(exact.abs().max())
            # the update is at most a few lr; its relative error is that of m and r where r is not tiny against the tensor's
            bound = HALF[dtype] * want.abs() + t * ulp * (want.abs() + 40 * HYPER['lr'])
            assert bool(((p.detach().double() - want).abs() <= bound * 1.01).all())
            m[i], v[i] = state['exp_avg'].double(), state['exp_avg_sq'].double()
        _regrad(params, g)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('max_norm', [None, 0.5])
def test_8_bit_steps_match_float64(dtype, max_norm):
    import spmm_cpp
    params, g = _params(SIZES, dtype, 2)
    opt = spmm_cpp.AdamW(params, state_bits=8, max_norm=max_norm, seed=5, **HYPER)
    for t in range(1, 6):
        _, coef = _coef(params, max_norm)
        before = [p.detach().double() for p in params]
        means = [_values(opt.state[p]) if p in opt.state else (torch.zeros_like(b), torch.zeros_like(b)) for p, b in zip(params, before)]
        opt.step()
        for p, b, (m0, r0) in zip(params, before, means):
            want, m, v = _step64(b, p.grad, m0, r0 * r0, t, coef)
            bound = HALF[dtype] * want.abs() + 16 * HALF[torch.float32] * (want.abs() + 40 * HYPER['lr'])
            assert bool(((p.detach().double() - want).abs() <= bound * 1.01).all())
            got_m, got_r = _values(opt.state[p])
            for got, exact in ((got_m, m), (got_r, v.sqrt())):
                step = torch.maximum(exact.abs() * 2.0 ** -3, _blocks_top(exact) * (2.0 ** -9 / 448))
                assert bool(((got - exact).abs() <= step * (1 + 1e-5)).all())
                assert bool((got * exact >= 0).all())
            assert bool((got_r[v > 0] > 0).all())
        _regrad(params, g)


def test_8_bit_rounding_has_no_bias():
    """A mean that stays where it is on average is kept on average: 4,096 equal numbers between two codes, 64 steps of their own gradient.  The sum
    of 4,096 roundings with a spread of at most half a step (2^-4) each has a standard deviation of 2^-4 / 64 / 2; six of them is 0.3 %.
    Rounded to nearest, all of them would be off by the same share of a step."""
    import spmm_cpp
    p = torch.nn.Parameter(torch.zeros(4096 + 16, device='cuda'))
    x = torch.full((4096 + 16,), 1.03, device='cuda')
    x[::257] = 1.9                                                 # one larger in every block, so that the others lie inside the grid
    opt = spmm_cpp.AdamW([p], lr=0.0, weight_decay=0.0, state_bits=8)
    for _ in range(64):
        p.grad = x.clone()
        opt.step()
    m, r = _values(opt.state[p])
    usual = x < 1.5
    assert abs(float(m[usual].mean()) / (1.03 * (1 - 0.9 ** 64)) - 1) < 0.01
    assert abs(float(r[usual].square().mean()) / (1.03 ** 2 * (1 - 0.999 ** 64)) - 1) < 0.03      # the square of a spread of 2^-5 adds 0.1 %


def test_8_bit_steps_repeat_and_depend_on_the_seed():
    import spmm_cpp
    out = []
    for seed in (3, 3, 4):
        params, g = _params(SIZES, torch.float32, 7)
        opt = spmm_cpp.AdamW(params, state_bits=8, seed=seed, **HYPER)
        for _ in range(3):
            opt.step()
            _regrad(params, g)
        out.append([t.view(torch.uint8) for p in params for t in (p.detach(), opt.state[p]['exp_avg'], opt.state[p]['root'])])
    assert all(torch.equal(a, b) for a, b in zip(out[0], out[1]))
    assert not all(torch.equal(a, b) for a, b in zip(out[0], out[2]))


@pytest.mark.parametrize('bits', [32, 8])
def test_many_tensors_views_and_gradients_with_strides(bits):
    """More tensors than one launch takes, of several types, at odd addresses, with gradients that are column slices of wider buffers: the same as one
    optimiser for each."""
    import spmm_cpp
    g = torch.Generator(device='cuda').manual_seed(3)
    params, alone = [], []
    for i in range(450):
        n = 1 + (i * 37) % 300
        dtype = (torch.float32, torch.bfloat16, torch.float16)[i % 3] if i % 50 == 0 else torch.float32
        base = torch.randn(n + 3, device='cuda', generator=g).to(dtype)
        p, q = torch.nn.Parameter(base[i % 3:i % 3 + n]), torch.nn.Parameter(base[i % 3:i % 3 + n].clone())
        wide = torch.randn(n, 2, device='cuda', generator=g).to(dtype)
        p.grad, q.grad = wide[:, 0], wide[:, 0].clone()
        params.append(p), alone.append(q)
    params[5].grad = alone[5].grad = None
    opt = spmm_cpp.AdamW([dict(params=params[:200]), dict(params=params[200:], lr=1e-2, betas=(0.8, 0.99))], state_bits=bits, **HYPER)
    untouched = params[5].detach().clone()
    for _ in range(2):
        opt.step()
    assert torch.equal(params[5], untouched) and int(opt.state[params[5]]['step']) == 0
    place = 0
    for i, (p, q) in enumerate(zip(params, alone)):
        if bits == 32 and q.grad is not None:                      # 8 bits: the place decides the noise
            one = spmm_cpp.AdamW([q], **(HYPER if i < 200 else dict(HYPER, lr=1e-2, betas=(0.8, 0.99))))
            one.step(), one.step()
            assert torch.equal(p, q) and torch.equal(opt.state[p]['exp_avg_sq'], one.state[q]['exp_avg_sq'])
        place += p.numel() + (-p.numel()) % 256
    assert all(bool(torch.isfinite(p).all()) for p in params)


@pytest.mark.parametrize('bits', [32, 8])
def test_state_survives_saving_and_copying(bits):
    import spmm_cpp
    params, g = _params(SIZES[:6], torch.bfloat16, 9)
    opt = spmm_cpp.AdamW(params, state_bits=bits, max_norm=1.0, seed=8, **HYPER)
    opt.step()
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    other = spmm_cpp.AdamW(twins, state_bits=bits, max_norm=1.0, seed=8)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    _regrad(params, g)
    for p, q in zip(params, twins):
        q.grad = p.grad.clone()
    opt.step(), other.step()
    for p, q in zip(params, twins):
        assert torch.equal(p, q)
        for name, value in opt.state[p].items():
            assert value.dtype == other.state[q][name].dtype and torch.equal(value.view(torch.uint8) if value.dim() else value, other.state[q][name].view(torch.uint8) if value.dim() else other.state[q][name])


def test_replaced_state_is_used():
    """What a program puts into the optimiser's state between two steps is what the next step reads and writes."""
    import spmm_cpp
    params, g = _params([(300,), (40,)], torch.float32, 4)
    opt = spmm_cpp.AdamW(params, **HYPER)
    opt.step()
    fresh = torch.zeros(300, device='cuda')
    old = opt.state[params[0]]['exp_avg']
    kept = old.clone()
    opt.state[params[0]]['exp_avg'] = fresh
    opt.step()
    assert torch.equal(old, kept) and float(fresh.abs().max()) > 0
    opt.state[params[1]] = dict(step=torch.tensor(41, device='cuda'), exp_avg=torch.zeros(40, device='cuda'), exp_avg_sq=torch.ones(40, device='cuda'))
    opt.step()
    assert int(opt.state[params[1]]['step']) == 42 and int(opt.state[params[0]]['step']) == 3
    with pytest.raises(RuntimeError, match='does not fit'):
        opt.state[params[1]]['exp_avg'] = torch.zeros(41, device='cuda')
        opt.step()


@pytest.mark.parametrize('bits', [32, 8])
def test_captured_steps_count_on(bits):
    """Three replays of a captured step, with new gradients in the captured buffers, are three eager steps."""
    import spmm_cpp
    params, g = _params(SIZES, torch.float32, 6)
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    for p, q in zip(params, twins):
        q.grad = p.grad.clone()
    opt, eager = (spmm_cpp.AdamW(ps, state_bits=bits, max_norm=0.7, **HYPER) for ps in (params, twins))
    opt.step(), eager.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(3):
        for p, q in zip(params, twins):
            p.grad.copy_(torch.randn(p.shape, device='cuda', generator=g))
            q.grad.copy_(p.grad)
        graph.replay()
        eager.step()
    for p, q in zip(params, twins):
        assert torch.equal(p, q) and int(opt.state[p]['step']) == 4
    assert torch.equal(opt.grad_norm, eager.grad_norm)


def test_on_another_stream_and_versions():
    import spmm_cpp
    params, _ = _params([(1000,)], torch.float32, 12)
    opt = spmm_cpp.AdamW(params, **HYPER)
    version = params[0]._version
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    assert params[0]._version > version                            # kept copies of a weight go by it
    assert int(opt.state[params[0]]['step']) == 1


@pytest.mark.parametrize('bits', [32, 8])
def test_non_finite_gradients_show(bits):
    import spmm_cpp
    p = torch.nn.Parameter(torch.ones(1000, device='cuda'))
    opt = spmm_cpp.AdamW([p], state_bits=bits, lr=1e-3)
    p.grad = torch.ones_like(p)
    p.grad[300], p.grad[700] = float('nan'), float('inf')
    opt.step()
    bad = ~torch.isfinite(p.detach())
    assert bad.nonzero().view(-1).tolist() == [300, 700]
    p.grad = torch.ones_like(p)
    opt.step()
    bad = ~torch.isfinite(p.detach())
    assert bool(bad[300]) and bool(bad[700]) and not bool(bad[:256].any())
    q = torch.nn.Parameter(torch.ones(10, device='cuda'))
    q.grad = torch.full_like(q, float('nan'))
    clipped = spmm_cpp.AdamW([q], max_norm=1.0)
    clipped.step()
    assert math.isnan(float(clipped.grad_norm)) and bool(torch.isnan(q.detach()).all())


def test_refusals():
    import spmm_cpp
    p = torch.nn.Parameter(torch.ones(4, 6, device='cuda'))
    opt = spmm_cpp.AdamW([p])
    p.grad = torch.ones(4, 6, device='cuda').to_sparse()
    with pytest.raises(RuntimeError, match='dense'):
        opt.step()
    q = torch.nn.Parameter(torch.ones(4, 6, device='cuda').t())
    q.grad = torch.ones(6, 4, device='cuda')
    with pytest.raises(RuntimeError, match='contiguous'):
        spmm_cpp.AdamW([q]).step()
    d = torch.nn.Parameter(torch.ones(4, device='cuda', dtype=torch.float64))
    with pytest.raises(RuntimeError, match='contiguous fp32'):
        spmm_cpp.AdamW([d]).step()
    opt = spmm_cpp.AdamW([p])
    p.grad = None
    opt.step()                                                     # nothing to do
    assert bool((p == 1).all())
    empty = torch.nn.Parameter(torch.empty(0, device='cuda'))
    empty.grad = torch.empty(0, device='cuda')
    spmm_cpp.AdamW([empty], max_norm=1.0).step()


def test_calls_that_would_go_wrong_are_refused():
    """Parameters that share elements (all are stepped at once), and a first step inside a capture (every replay would start anew)."""
    import spmm_cpp
    base = torch.ones(100, device='cuda')
    a, b = torch.nn.Parameter(base[:60]), torch.nn.Parameter(base[59:])
    a.grad, b.grad = torch.ones(60, device='cuda'), torch.ones(41, device='cuda')
    with pytest.raises(RuntimeError, match='share memory'):
        spmm_cpp.AdamW([a, b]).step()
    b = torch.nn.Parameter(base[60:])
    b.grad = torch.ones(40, device='cuda')
    opt = spmm_cpp.AdamW([a, b])
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match='before capturing'):
        with torch.cuda.graph(graph, stream=stream):
            opt.step()
    opt.step()
    assert float(base.max()) < 1


def test_schedulers_hooks_and_foreign_state():
    """A learning rate that a scheduler sets is the next step's; hooks run; the state of torch.optim.AdamW over fp32 parameters can be taken over."""
    import spmm_cpp
    params, g = _params([(300,), (7, 5)], torch.float32, 21)
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    opt, ref = spmm_cpp.AdamW(params, **HYPER), torch.optim.AdamW(twins, foreach=False, **HYPER)
    seen = []
    handle = opt.register_step_post_hook(lambda *args: seen.append(1))
    schedulers = [torch.optim.lr_scheduler.StepLR(o, 2, 0.1) for o in (opt, ref)]
    for t in range(5):
        for p, q in zip(params, twins):
            q.grad = p.grad.clone()
        opt.step(), ref.step()
        [s.step() for s in schedulers]
        if t == 2:
            handle.remove()
        _regrad(params, g)
    assert len(seen) == 3 and opt.param_groups[0]['lr'] == ref.param_groups[0]['lr'] < HYPER['lr']
    for p, q in zip(params, twins):                                # five steps of rates up to 3e-3, each within 2^-19 of itself, on numbers of order one
        assert float((p - q).abs().max()) <= 5 * (2.0 ** -19 * 40 * HYPER['lr'] + 2.0 ** -23 * float(q.abs().max()))
    other = spmm_cpp.AdamW([torch.nn.Parameter(q.detach().clone()) for q in twins])
    other.load_state_dict(ref.state_dict())
    heirs = other.param_groups[0]['params']
    for p, q in zip(heirs, twins):
        p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    other.step(), ref.step()
    assert int(other.state[heirs[0]]['step']) == 6
    for p, q in zip(heirs, twins):
        assert float((p - q).abs().max()) <= 2.0 ** -19 * 40 * HYPER['lr'] + 2.0 ** -22 * float(q.abs().max())


def test_norm_of_no_gradients_in_a_replayed_graph():
    """Entries without elements: the norm is 0 and the factor 1, in a graph too, which holds nothing of the call's own stack."""
    import ctypes
    import spmm_cpp
    lib, empty = spmm_cpp.lib(), (ctypes.c_char * 512)()      # zeroed entries: n == 0
    lib.dg_adamw_workspace.restype = ctypes.c_int64
    size = lib.dg_adamw_workspace(empty, ctypes.c_int32(1))
    workspace, result = torch.zeros(size, dtype=torch.uint8, device='cuda'), torch.empty(2, device='cuda')

    def norm():
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        assert lib.dg_grad_norm(empty, ctypes.c_int32(1), ctypes.c_double(2.0), ctypes.c_void_p(result.data_ptr()), ctypes.c_void_p(workspace.data_ptr()),
                                ctypes.c_int64(size), stream) == 0
    norm()
    assert result.tolist() == [0.0, 1.0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm()
    result.fill_(7.0)
    graph.replay()
    assert result.tolist() == [0.0, 1.0]


@pytest.mark.parametrize('bits', [32, 8])
def test_gradients_whose_square_overflows_show(bits):
    import spmm_cpp
    p = torch.nn.Parameter(torch.ones(600, device='cuda'))
    p.grad = torch.zeros_like(p)
    p.grad[300] = 1e20
    opt = spmm_cpp.AdamW([p], state_bits=bits)
    opt.step()
    assert torch.isnan(p[300]) and torch.isfinite(p[:256]).all() and torch.isfinite(p[512:]).all()
