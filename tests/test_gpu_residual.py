"""The residual GCN - Aggregate, spmm_cpp.linear with bias, activation and residual, spmm_cpp.AdamW - as training uses them together, against float64.
Needs a GPU."""
import math
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def env1():
    from dist_utils import DistEnv
    os.environ.setdefault('MASTER_ADDR', '127.0.0.1')
    os.environ['MASTER_PORT'] = '29747'
    os.environ.setdefault('DIST_GNN_LOG_ROOT', '/tmp/dist_gnn_test_logs')
    env = DistEnv(0, 1, 'nccl')
    yield env
    env.shutdown()


def _graph(nodes, feat, classes, seed=3):
    """A random symmetric graph, normalised, with features and labels, as the loaders hand it over."""
    from coo_graph import COO_Graph, Parted_COO_Graph
    gen = torch.Generator().manual_seed(seed)
    pairs = torch.randint(0, nodes, (2, 6 * nodes), generator=gen)
    pairs = pairs[:, pairs[0] != pairs[1]]
    edges = torch.unique(torch.cat([pairs, pairs.flip(0)], 1), dim=1)
    mask = torch.rand(nodes, generator=gen)
    data = dict(edge_index=edges, features=torch.randn(nodes, feat, generator=gen), labels=torch.randint(0, classes, (nodes,), generator=gen),
                train_mask=mask < 0.6, val_mask=(mask >= 0.6) & (mask < 0.8), test_mask=mask >= 0.8, num_nodes=nodes, num_edges=edges.size(1), num_classes=classes)
    full = COO_Graph.from_dict('residual', data, device='cuda')
    return Parted_COO_Graph.from_full(full, 0, 1)


def _dense(g):
    a = g.adj_parts[0]
    return torch.sparse_coo_tensor(a.indices(), a.values().double(), a.shape).to_dense()


def _forward64(A, x, weights, biases, act):
    h = x.double()
    for l, (w, b) in enumerate(zip(weights, biases)):
        z = A @ h @ w + b
        if l == len(weights) - 1:
            return z
        cdf = 0.5 * torch.erfc(-z * math.sqrt(0.5))
        value = z.clamp(min=0) if act == 'relu' else z * cdf if act == 'gelu' else z * torch.sigmoid(z)
        h = value + h if l > 0 else value


def _small(model, gen):
    """Weights of a usual initialiser and biases that are not zero."""
    with torch.no_grad():
        for name, p in model.named_parameters():
            p.copy_(torch.randn(p.shape, device='cuda', generator=gen) * (p.size(0) ** -0.5 if p.dim() == 2 else 0.3))


@pytest.mark.parametrize('nodes,feat,hidden,classes,layers,act', [(700, 24, 32, 7, 3, 'gelu'), (1500, 33, 64, 10, 4, 'silu'), (300, 16, 20, 5, 2, 'gelu'), (9, 5, 8, 3, 4, 'silu')])
def test_outputs_and_gradients_match_float64(env1, nodes, feat, hidden, classes, layers, act):
    """Every product is within 1e-5 of its largest element (tests of the products themselves); a chain of `layers` of them, forward and backward, of that
    times their number."""
    from models import GCN
    g = _graph(nodes, feat, classes)
    model = GCN(g, env1, hidden_dim=hidden, num_layers=layers, bias=True, residual=True, activation=act)
    gen = torch.Generator(device='cuda').manual_seed(1)
    _small(model, gen)
    out = model(g.features)
    c = torch.randn(out.shape, device='cuda', generator=gen)
    out.backward(c)
    weights = [w.detach().double().requires_grad_() for w in model.weights()]
    biases = [getattr(model, f'bias{l + 1}').detach().double().requires_grad_() for l in range(layers)]
    want = _forward64(_dense(g), g.features, weights, biases, act)
    want.backward(c.double())
    tol = 1e-5 * 2 * layers
    assert float((out.detach().double() - want).abs().max()) <= tol * float(want.abs().max())
    for l in range(layers):
        for mine, exact in ((model.weights()[l].grad, weights[l].grad), (getattr(model, f'bias{l + 1}').grad, biases[l].grad)):
            assert float((mine.double() - exact).abs().max()) <= tol * float(exact.abs().max()), l


@pytest.mark.parametrize('optimizer', ['adamw', 'adamw8'])
def test_training_runs_and_steps_match_float64(env1, optimizer):
    """Three epochs of dist_train.train.  The first step's weights: AdamW's first step is lr times the gradient's sign, whatever its size (but for eps, 1e-8),
    so where a gradient is larger than its error the step is known to the rounding of p and of about ten operations."""
    import dist_train
    import spmm_cpp
    from models import GCN
    g = _graph(800, 24, 6)
    model, losses = dist_train.train(g, env1, total_epoch=3, hidden_dim=32, num_layers=4, optimizer=optimizer, bias=True, residual=True, activation='gelu')
    assert len(losses) == 3 and all(math.isfinite(v) for v in losses)
    assert {name for name, _ in model.named_parameters()} == {f'{k}{l}' for k in ('weight', 'bias') for l in range(1, 5)}
    model = GCN(g, env1, hidden_dim=32, num_layers=4, bias=True, residual=True, activation='gelu')
    gen = torch.Generator(device='cuda').manual_seed(1)
    _small(model, gen)
    opt = dist_train.make_optimizer(optimizer, model.parameters())
    assert isinstance(opt, spmm_cpp.AdamW)
    before = {name: p.detach().double() for name, p in model.named_parameters()}
    loss = dist_train.local_loss(g, model(g.features), torch.nn.CrossEntropyLoss())
    loss.backward()
    weights = [before[f'weight{l}'].clone().requires_grad_() for l in range(1, 5)]
    biases = [before[f'bias{l}'].clone().requires_grad_() for l in range(1, 5)]
    rows = g.local_train_mask
    want = torch.nn.functional.cross_entropy(_forward64(_dense(g), g.features, weights, biases, 'gelu')[rows], g.local_labels[rows])
    want.backward()
    assert abs(float(loss) - float(want)) <= 1e-4 * float(want)
    opt.step()
    for l in range(1, 5):
        for name, exact in ((f'weight{l}', weights[l - 1].grad), (f'bias{l}', biases[l - 1].grad)):
            p = dict(model.named_parameters())[name].detach().double()
            sure = exact.abs() > 1e-3 * exact.abs().max()
            moved = before[name] * (1 - 0.01 * 0.01) - 0.01 * exact.sign() * (exact.abs() / (exact.abs() + 1e-8))
            error = 0.1 * 1e-8 / exact.abs().clamp(min=1e-12) + 2.0 ** -19         # eps beside a gradient that is a tenth off, and the operations
            assert bool(((p - moved).abs() <= 0.01 * error + 2.0 ** -23 * before[name].abs())[sure].all())


def test_plain_layers_equal_the_fused_network(env1):
    """bias, all zero, changes the path and not the result beyond rounding: Aggregate and linear against DistGCNLayer."""
    from models import GCN
    g = _graph(600, 24, 6)
    gen = torch.Generator(device='cuda').manual_seed(5)
    weights = [torch.randn(a, b, device='cuda', generator=gen) * a ** -0.5 for a, b in ((24, 32), (32, 32), (32, 6))]
    plain, biased = GCN(g, env1, hidden_dim=32, weights=weights), GCN(g, env1, hidden_dim=32, weights=weights, bias=True)
    a, b = plain(g.features), biased(g.features)
    assert float((a - b).abs().max()) <= 2e-5 * float(a.abs().max())
    a.sum().backward(), b.sum().backward()
    for p, q in zip(plain.weights(), biased.weights()):
        assert float((p.grad - q.grad).norm()) <= 1e-4 * float(p.grad.norm())


def test_options_that_do_not_go_together():
    from models import GCN
    for bad in (dict(bias=True, cache_input_product=True), dict(residual=True, transform_first=True), dict(activation='gelu', input_gradient_shortcut=True),
                dict(activation='tanh')):
        with pytest.raises(ValueError):
            GCN(None, None, **bad)
