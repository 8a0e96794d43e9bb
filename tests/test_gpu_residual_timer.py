"""The timer's regions in a step of the residual GCN.  Needs a GPU."""
import pytest
import torch

from test_gpu_residual import _graph, env1          # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def test_products_are_timed_in_both_passes(env1):          # noqa: F811
    """As many regions as the plain layers have: a product forward and one region backward a layer, each of some length."""
    from models import GCN
    g = _graph(5000, 64, 16)
    counts, times = {}, {}
    for kind, options in (('plain', {}), ('residual', dict(bias=True, residual=True, activation='gelu'))):
        model = GCN(g, env1, hidden_dim=128, num_layers=3, **options)
        for _ in range(2):
            env1.timer.resolve()
            before = env1.timer.count_dict['mm'], env1.timer.duration_dict['mm']
            out = model(g.features)
            env1.timer.resolve()
            forward = env1.timer.count_dict['mm'], env1.timer.duration_dict['mm']
            out.backward(torch.ones_like(out))
            env1.timer.resolve()
            after = env1.timer.count_dict['mm'], env1.timer.duration_dict['mm']
        counts[kind] = forward[0] - before[0], after[0] - forward[0]
        times[kind] = forward[1] - before[1], after[1] - forward[1]
    assert counts['residual'] == (3, 3) == counts['plain']
    assert min(times['residual']) > 0
