"""Host logic of the residual GCN's layers: weights whose gradients are summed over the ranks, on CPU with a stand-in for the environment."""
import contextlib

import torch


class _Timer:
    def timing_cuda(self, tag):
        return contextlib.nullcontext()

    def empty_region(self, tag):
        pass


class _Env:
    def __init__(self, world_size):
        self.world_size, self.timer, self.sums = world_size, _Timer(), 0

    def all_reduce_sum(self, t):
        self.sums += 1
        t.mul_(self.world_size)


def test_gradients_of_shared_weights_are_summed_once(monkeypatch):
    from dist_utils import DistEnv
    from models import gcn
    for world in (1, 4):
        env = _Env(world)
        monkeypatch.setattr(DistEnv, 'env', env, raising=False)
        w = torch.randn(5, 3, requires_grad=True)
        up = torch.randn(5, 3)
        kept = up.clone()
        (gcn.SumOverRanks.apply(w) * 1.0).backward(up)
        assert torch.equal(w.grad, up * world) and torch.equal(up, kept) and env.sums == (world > 1)
        x = torch.ones(3, requires_grad=True)
        gcn.SumOverRanks.apply(x).sum().backward()                   # an expanded gradient
        assert torch.equal(x.grad, torch.full((3,), float(world)))


def test_backward_of_an_operation_is_timed():
    """One region from before its node to behind it, for every backward pass; none where nothing is differentiated."""
    from models import gcn
    events = []

    class Region:
        def __enter__(self):
            events.append('enter')
            return self

        def __exit__(self, *exc):
            events.append('leave')

    class Timer:
        def timing_cuda(self, tag):
            assert tag == 'mm'
            return Region()

    w = torch.ones(3, 2, requires_grad=True)
    x = torch.ones(4, 3, requires_grad=True)
    x.register_hook(lambda g: events.append('x'))
    y = gcn._time_backward(x @ w, Timer())
    (y * 2).sum().backward(retain_graph=True)
    assert events == ['enter', 'leave', 'x']
    (y * 2).sum().backward()
    assert events == ['enter', 'leave', 'x'] * 2
    gcn._time_backward(x.detach() @ w.detach(), Timer())
