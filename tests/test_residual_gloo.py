"""The residual GCN on several ranks: every rank's rows of the outputs and the weights' and biases' gradients, summed over the ranks, against the whole graph in one piece.
CPU ranks over gloo; the sparse product, the exchange and the linear layer are done by the test, in float64 - the product has no CPU engine."""
import os
import sys
import tempfile

import numpy as np
import pytest
import torch

from conftest import PKG, ROOT


def _act(name, z):
    return torch.relu(z) if name == 'relu' else torch.nn.functional.gelu(z) if name == 'gelu' else torch.nn.functional.silu(z) if name == 'silu' else z


def _linear(x, weight, bias=None, residual=None, activation=None):
    z = x @ weight + (0 if bias is None else bias)
    return _act(activation, z) + (0 if residual is None else residual)


def _graph(nodes, feat, classes):
    gen = torch.Generator().manual_seed(nodes)
    pairs = torch.randint(0, nodes, (2, 5 * nodes), generator=gen)
    pairs = pairs[:, pairs[0] != pairs[1]]
    edges = torch.unique(torch.cat([pairs, pairs.flip(0)], 1), dim=1)
    mask = torch.rand(nodes, generator=gen)
    return dict(edge_index=edges, features=torch.randn(nodes, feat, generator=gen), labels=torch.randint(0, classes, (nodes,), generator=gen), train_mask=mask < 0.6,
                val_mask=(mask >= 0.6) & (mask < 0.8), test_mask=mask >= 0.8, num_nodes=nodes, num_edges=edges.size(1), num_classes=classes)


def _worker(rank, world, port, out_dir, options, shape):
    os.environ.update(MASTER_ADDR='127.0.0.1', MASTER_PORT=str(port), DIST_GNN_LOG_ROOT=out_dir)
    for p in (ROOT, PKG):
        if p not in sys.path:
            sys.path.insert(0, p)
    import torch.distributed as dist
    import spmm_cpp
    from coo_graph import COO_Graph, Parted_COO_Graph
    from dist_utils import DistEnv
    from models import GCN, gcn
    torch.set_num_threads(1)
    env = DistEnv(rank, world, 'gloo')
    try:
        full = COO_Graph.from_dict('residual', _graph(*shape[:3]), device=env.device)
        g = Parted_COO_Graph.from_full(full, rank, world)
        blocks = [torch.sparse_coo_tensor(a.indices(), a.values().double(), a.shape).to_dense() for a in g.adj_parts]

        def product(adj_parts, x, constant=False):
            z = torch.zeros(blocks[0].size(0), x.size(1), dtype=torch.float64)
            for st in env.stages():
                buf = x.detach().contiguous().clone() if st.root_global == rank else torch.empty(blocks[st.part].size(1), x.size(1), dtype=torch.float64)
                dist.broadcast(buf, src=st.root_global)
                z += blocks[st.part] @ buf
            return z

        gcn._distributed_spmm, spmm_cpp.linear = product, _linear
        gen = torch.Generator().manual_seed(7)
        model = GCN(g, env, hidden_dim=shape[3], num_layers=shape[4], **options).double()
        with torch.no_grad():
            for p in model.parameters():
                p.copy_(torch.randn(p.shape, generator=gen, dtype=torch.float64) * (p.size(0) ** -0.5 if p.dim() == 2 else 0.3))
        x = g.features.double()
        out = model(x)
        c = torch.randn(out.shape, generator=torch.Generator().manual_seed(100 + rank), dtype=torch.float64)
        out.backward(c)
        rec = dict(A=torch.cat(blocks, 1).numpy(), x=x.numpy(), c=c.numpy(), out=out.detach().numpy())
        for name, p in model.named_parameters():
            rec['p/' + name], rec['g/' + name] = p.detach().numpy(), p.grad.numpy()
        np.savez(os.path.join(out_dir, f'rank{rank}.npz'), **rec)
    finally:
        env.shutdown()


@pytest.mark.parametrize('world,options,shape', [(2, dict(bias=True, residual=True, activation='gelu'), (41, 6, 5, 8, 4)), (3, dict(residual=True, activation='silu'), (50, 9, 3, 7, 3)),
                                                 (2, dict(bias=True), (24, 5, 4, 6, 2))])
def test_ranks_together_are_the_whole_graph(world, options, shape):
    import torch.multiprocessing as mp
    out_dir = tempfile.mkdtemp(prefix='dg_residual_')
    mp.spawn(_worker, (world, 29861 + world, out_dir, options, shape), nprocs=world, join=True)
    ranks = [np.load(os.path.join(out_dir, f'rank{r}.npz')) for r in range(world)]
    A, x, c = (torch.from_numpy(np.concatenate([r[k] for r in ranks])) for k in 'Axc')
    assert torch.equal(A, A.t())                                    # what Aggregate's backward takes for granted
    params = {k[2:]: torch.from_numpy(ranks[0][k]).requires_grad_() for k in ranks[0].files if k.startswith('p/')}
    act, layers = options.get('activation', 'relu'), shape[4]
    h = x
    for l in range(1, layers + 1):
        last = l == layers
        y = _linear(A @ h, params[f'weight{l}'], params.get(f'bias{l}'), activation=None if last else act)
        h = y + h if options.get('residual') and 1 < l < layers else y
    h.backward(c)
    at = 0
    for r in ranks:
        rows = r['out'].shape[0]
        assert np.abs(r['out'] - h.detach().numpy()[at:at + rows]).max() <= 1e-12 * max(1.0, float(h.abs().max()))
        at += rows
        for name, p in params.items():
            assert np.array_equal(r['p/' + name], p.detach().numpy())
            assert np.abs(r['g/' + name] - p.grad.numpy()).max() <= 1e-12 * max(1.0, float(p.grad.abs().max())), name
