"""Activations of spmm_cpp.linear over the whole range of their types, through every kernel that computes them, against float64.  Needs a GPU.

The layers here have one input and weights or inputs of one, so that z is the number itself: in 16 bits exactly, in fp32 by three TF32 passes to 2^-21 of it.
Tolerances.  HALF is half a step of the type.  GELU is z - |z| Phi(-|z|) or - |z| Phi(-|z|): the formula's share of the tail, 2e-5 where two elements are taken at a
time (16 bits, many rows), 1.2e-6 elsewhere, and that of the exponential's argument, z^2 2^-24.  SiLU: (|z| + 16) 2^-24 of the value, and where two are taken at a
time the sigmoid stands at 2^-60 below -41.6, z at -60: 6e-17.  Slopes add the rounding of sums of numbers of order one, (min(|z|, 60) + 16) 2^-23.  What lies below
the type's smallest normal number is off by 2^-25 (fp16), or 2^-120."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
FLOOR = {torch.float32: 2.0 ** -120, torch.bfloat16: 2.0 ** -120, torch.float16: 2.0 ** -25}


def _grid(dtype):
    top = torch.finfo(dtype).max
    far = torch.logspace(-6, math.log10(top) - 0.001, 700, dtype=torch.float64)
    near = torch.linspace(-16, 16, 2001, dtype=torch.float64)
    border = torch.tensor([0.0, 41.5, 41.7, 42.0, 59.5, 60.5, 87.0, 89.0, 104.0, top], dtype=torch.float64)
    z = torch.cat([far, -far, near, border, -border])
    z = z[torch.randperm(z.numel(), generator=torch.Generator().manual_seed(1))]      # neighbours of every size, two of which go together
    return z.to(dtype).cuda()


def _exact(act, z):
    """value, slope, and the tail of a bell that errors are measured by, in float64"""
    z = z.double()
    if act == 'silu':
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s)), s.new_zeros(())
    cdf, bell = 0.5 * torch.erfc(-z * math.sqrt(0.5)), torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return z * cdf, cdf + z * bell, 0.5 * torch.erfc(z.abs() * math.sqrt(0.5))


def _bounds(act, z, dtype, pairs):
    value, slope, tail = _exact(act, z)
    a, half, near = z.double().abs(), HALF[dtype], z.double().abs().clamp(max=16)
    moved = 2.0 ** -21 * a * slope.abs() if dtype == torch.float32 else torch.zeros_like(a)      # z itself
    if act == 'gelu':
        share = (2e-5 if pairs else 1.2e-6) + near ** 2 * 2.0 ** -24
        ev = share * a * tail + 2.0 ** -23 * value.abs()
        es = share * (tail + a * torch.exp(-0.5 * a * a)) + 2.0 ** -22 * slope.abs().clamp(max=1.2)
        moved_slope = 2.0 ** -21 * a * torch.exp(-0.5 * a * a) * (2 + a * a)
    else:
        ev = (a.clamp(max=104) + 16) * 2.0 ** -24 * value.abs() + (6e-17 if pairs else 0.0)
        es = (a.clamp(max=60) + 16) * 2.0 ** -23 * torch.where(z > 0, slope, slope.abs() + torch.sigmoid(z.double())) + (6e-17 if pairs else 0.0)
        moved_slope = 2.0 ** -21 * a * torch.exp(-a) * (2 + a)
    if dtype != torch.float32:
        moved_slope = torch.zeros_like(a)
    by_value = half * value.abs() + 1.01 * (ev + moved) + FLOOR[dtype] * (1 + near)
    by_slope = half * slope.abs() + 1.01 * (es + moved_slope) + 2.0 ** -21 * slope.abs() * (dtype == torch.float32) + FLOOR[dtype] * (1 + near)
    return value, slope, by_value, by_slope


def _within(got, want, bound, z, what):
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), (what, [(float(z[i]), float(got[i]), float(want[i])) for i in bad.nonzero().view(-1)[:5]])


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('act', ['gelu', 'silu'])
@pytest.mark.parametrize('form', ['many', 'panels', 'few', 'narrow'])
def test_values_over_the_whole_range(form, act, dtype):
    import spmm_cpp
    z = _grid(dtype)
    pairs = dtype != torch.float32 and form in ('many', 'panels')
    value, _, bound, _ = _bounds(act, z, dtype, pairs)
    if form in ('many', 'narrow'):                                 # z down a column of x
        y = spmm_cpp.linear(z[:, None], torch.ones(1, 48 if form == 'many' else 8, device='cuda', dtype=dtype), activation=act)
        assert bool((y == y[:, :1]).all())
        y = y[:, 0]
    else:                                                          # z along a row of the weight
        y = spmm_cpp.linear(torch.ones(40 if form == 'panels' else 3, 1, device='cuda', dtype=dtype), z[None], activation=act)
        assert bool((y == y[:1]).all())
        y = y[0]
    _within(y, value, bound, z, 'value')
    assert spmm_cpp.dense_status() == 0


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('act', ['gelu', 'silu'])
@pytest.mark.parametrize('form', ['back', 'alone', 'few', 'narrow'])
def test_slopes_over_the_whole_range(form, act, dtype):
    """One column (row) of the incoming gradient is one, the others are zero: x's (w's) gradient is the slope."""
    import spmm_cpp
    z = _grid(dtype)
    _, slope, _, bound = _bounds(act, z, dtype, dtype != torch.float32 and form != 'narrow')
    if form == 'few':
        x, w = torch.ones(3, 1, device='cuda', dtype=dtype), z[None].clone().requires_grad_()
        dy = torch.zeros(3, z.numel(), device='cuda', dtype=dtype)
        dy[0] = 1
        got = torch.autograd.grad(spmm_cpp.linear(x, w, activation=act), w, dy)[0][0]
    else:
        N = 8 if form == 'narrow' else 48
        x, w = z[:, None].clone().requires_grad_(), torch.ones(1, N, device='cuda', dtype=dtype, requires_grad=form != 'alone')
        dy = torch.zeros(z.numel(), N, device='cuda', dtype=dtype)
        dy[:, 0] = 1
        got = torch.autograd.grad(spmm_cpp.linear(x, w, activation=act), [x, w] if form != 'alone' else [x], dy)[0][:, 0]
    _within(got, slope, bound, z, 'slope')
    assert spmm_cpp.dense_status() == 0


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('act', ['gelu', 'silu'])
def test_what_is_not_a_number_stays_one(act, dtype):
    """In every form, value and slope, whatever stands beside it."""
    import spmm_cpp
    for N, M in ((48, 400), (48, 3), (8, 400)):
        x = torch.full((M, 1), -50.0, device='cuda', dtype=dtype)
        x[1], x[2] = float('nan'), 100.0
        for asked in ('x', 'xw'):
            a, w = x.clone().requires_grad_(), torch.ones(1, N, device='cuda', dtype=dtype, requires_grad=asked == 'xw')
            y = spmm_cpp.linear(a, w, activation=act)
            dx = torch.autograd.grad(y, [a] + [w] * (asked == 'xw'), torch.ones_like(y))[0]
            assert bool(torch.isnan(y[1]).all()) and bool(torch.isfinite(y[0]).all()) and bool(torch.isfinite(y[2:]).all())
            assert bool(torch.isnan(dx[1])) and bool(torch.isfinite(dx[0])) and bool(torch.isfinite(dx[2:]).all())
