"""spmm_cpp.AdamW where numbers are very small, in forms that its other tests leave out, against the formula in float64.  Needs a GPU."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('bits', [32, 8])
def test_second_means_below_the_normal_numbers(bits):
    """Gradients whose mean square is one of fp32's subnormal numbers, without eps: the step is lr m / sqrt(v) of those numbers, v = (1 - b2) g^2 as fp32 rounds it (one
    operation after the other).  The root is within 2^-22, the reciprocals and the other operations within 2^-20; p is zero before, so nothing is lost beside it."""
    import spmm_cpp
    g = torch.logspace(-21.5, -15, 4096, device='cuda', dtype=torch.float64).float()
    g[1::2] *= -1
    p = torch.nn.Parameter(torch.zeros_like(g))
    p.grad = g.clone()
    opt = spmm_cpp.AdamW([p], lr=1e-2, eps=0.0, weight_decay=0.0, state_bits=bits)
    opt.step()
    v = (g * g) * torch.tensor(1 - 0.999, dtype=torch.float32, device='cuda')
    some = v > 0                                                   # (1 - b2) g^2 is zero in fp32 below g = 1e-21
    assert int((some & (v < 2.0 ** -126)).sum()) > 500
    if bits == 32:
        assert torch.equal(opt.state[p]['exp_avg_sq'], v)
    m = torch.tensor(1 - 0.9, dtype=torch.float32).double().cuda() * g.double()
    want = -1e-2 / (1 - 0.9) * m / (v.double().sqrt() / math.sqrt(1 - 0.999))
    off = ((p.detach().double() - want).abs() / want.abs())[some]
    assert float(off.max()) <= 2.0 ** -20, (float(off.max()), float(g[some][off.argmax()]))


@pytest.mark.parametrize('bits', [32, 8])
def test_a_captured_step_keeps_what_it_writes(bits):
    """A graph of a step replayed after the optimiser has taken over another state and a group more: it steps the state of the capture, and no memory that has been given
    out since changes."""
    import copy
    import spmm_cpp
    params = [torch.nn.Parameter(torch.randn(n, device='cuda')) for n in (5000, 300, 7)]
    for p in params:
        p.grad = torch.randn_like(p)
    opt = spmm_cpp.AdamW(params, state_bits=bits, max_norm=1.0)
    opt.step()
    saved = copy.deepcopy(opt.state_dict())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    held = [(opt.state[p]['step'], opt.state[p]['exp_avg']) for p in params]
    opt.load_state_dict(saved)
    opt.step()                                                     # with the loaded state
    more = torch.nn.Parameter(torch.randn(9, device='cuda'))
    more.grad = torch.ones_like(more)
    opt.add_param_group(dict(params=[more]))
    opt.step()
    loaded = [opt.state[p]['exp_avg'].clone() for p in params]
    fresh = [torch.full((n,), 77, dtype=torch.uint8, device='cuda') for n in (512, 1024, 4096, 20_000, 40_000, 400_000) for _ in range(40)]
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert [int(step) for step, _ in held] == [2 + k] * 3
    assert all(bool((t == 77).all()) for t in fresh)
    assert [int(opt.state[p]['step']) for p in params] == [3, 3, 3] and int(opt.state[more]['step']) == 1
    assert all(torch.equal(a.view(torch.uint8), opt.state[p]['exp_avg'].view(torch.uint8)) for a, p in zip(loaded, params))
    opt.step()
    assert [int(opt.state[p]['step']) for p in params] == [4, 4, 4]


def test_8_bit_steps_over_many_tensors_match_float64():
    """More tensors than one launch takes, of three types, at odd addresses, with gradients that are column slices of wider buffers: every one's step, codes and scales,
    against the formula, from the means that the codes stand for.  Bounds: a parameter rounds by half a step of its type beside sixteen of fp32; a mean moves to a
    neighbour, at most one step of e4m3, 2^-3 of the value or 2^-9 / 448 of its block's largest."""
    import spmm_cpp
    half = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
    g = torch.Generator(device='cuda').manual_seed(3)
    params = []
    for i in range(450):
        n = 1 + (i * 37) % 300 + (2048 if i % 60 == 7 else 0)
        dtype = (torch.float32, torch.bfloat16, torch.float16)[i % 3]
        p = torch.nn.Parameter(torch.randn(n + 3, device='cuda', generator=g).to(dtype)[i % 3:i % 3 + n])
        params.append(p)

    def regrad():
        for i, p in enumerate(params):
            p.grad = torch.randn(p.numel(), 2, device='cuda', generator=g).to(p.dtype)[:, i % 2] * 10.0 ** -(i % 4)

    def values(state):
        return [(state[name].float().double() * state[name + '_scale'].double().repeat_interleave(256)[:state[name].numel()]) for name in ('exp_avg', 'root')]

    def top(x):
        flat = torch.zeros(x.numel() + (-x.numel()) % 256, dtype=torch.float64, device='cuda')
        flat[:x.numel()] = x.abs()
        return flat.view(-1, 256).amax(1).repeat_interleave(256)[:x.numel()]

    groups = [dict(params=params[:200]), dict(params=params[200:], lr=1e-2, betas=(0.8, 0.99))]
    opt = spmm_cpp.AdamW(groups, lr=3e-3, weight_decay=0.05, state_bits=8)
    for t in (1, 2, 3):
        regrad()
        before = [p.detach().double() for p in params]
        means = [values(opt.state[p]) if p in opt.state else [torch.zeros_like(b), torch.zeros_like(b)] for p, b in zip(params, before)]
        opt.step()
        for i, p in enumerate(params):
            lr, (b1, b2) = (3e-3, (0.9, 0.999)) if i < 200 else (1e-2, (0.8, 0.99))
            grad, (m, r) = p.grad.double(), means[i]
            m, v = b1 * m + (1 - b1) * grad, b2 * r * r + (1 - b2) * grad * grad
            want = before[i] * (1 - lr * 0.05) - lr * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + 1e-8)
            bound = half[p.dtype] * want.abs() + 16 * half[torch.float32] * (want.abs() + 40 * lr)
            assert bool(((p.detach().double() - want).abs() <= bound * 1.01).all()), i
            for got, exact in zip(values(opt.state[p]), (m, v.sqrt())):
                step = torch.maximum(exact.abs() * 2.0 ** -3, top(exact) * (2.0 ** -9 / 448))
                assert bool(((got - exact).abs() <= step * (1 + 1e-5)).all()) and bool((got * exact >= 0).all()), i
