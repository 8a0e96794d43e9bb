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
