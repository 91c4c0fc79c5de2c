"""GCN layers with bias, activation and skip connection in their product, on the GPU through the HIP kernels: against their
formulas in 64 bits, and train() with the optimisers of build_optimizer."""
import os
import socket

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _raw(g, dev):
    return {"edge_index": torch.from_numpy(g['edge_index']).to(dev), "features": torch.from_numpy(g['raw_features']).to(dev),
            "labels": torch.from_numpy(g['labels']).to(dev), "train_mask": torch.from_numpy(g['train_mask']).to(dev),
            "val_mask": torch.from_numpy(g['val_mask']).to(dev), "test_mask": torch.from_numpy(g['test_mask']).to(dev),
            "num_nodes": int(g['num_nodes']), "num_edges": g['edge_index'].shape[1], "num_classes": int(g['num_classes'])}


@pytest.fixture(scope='module')
def env(tmp_path_factory):
    import torch.distributed as dist
    import dist_utils
    with socket.socket() as s:
        s.bind(('127.0.0.1', 0))
        port = s.getsockname()[1]
    os.environ.update(MASTER_ADDR='127.0.0.1', MASTER_PORT=str(port), DGNN_LOG_DIR=str(tmp_path_factory.mktemp('logs')))
    e = dist_utils.DistEnv(0, 1, 'nccl', echo=False)
    assert e.device.type == 'cuda'
    yield e
    dist.destroy_process_group()


def _graph(env, golden_dir, name):
    import coo_graph
    g = np.load(os.path.join(golden_dir, f'{name}_graph.npz'))
    full = coo_graph.COO_Graph(name, attr_dict=_raw(g, env.device), device=env.device)
    return coo_graph.Parted_COO_Graph(name, 0, 1, device=env.device, attr_dict=full.partition(1, save=False)[0])


def _act(t, act):
    return {'none': lambda: t, 'relu': lambda: torch.relu(t), 'gelu': lambda: torch.nn.functional.gelu(t),
            'silu': lambda: torch.nn.functional.silu(t)}[act]()


@pytest.mark.parametrize('act', ['none', 'relu', 'gelu', 'silu'])
@pytest.mark.parametrize('skip', [False, True])
def test_layer_matches_its_formulas(env, golden_dir, act, skip):
    """1e-5 of each result's largest value, the project's bar for fp32 layers; relu is met away from its corner."""
    from models import gcn
    g = _graph(env, golden_dir, 'ragged')
    n = g.features.size(0)
    gen = torch.Generator(device='cuda').manual_seed(5)
    x, w, b, dy = (torch.randn(*s, generator=gen, device='cuda') for s in ((n, 24), (24, 24), (24,), (n, 24)))
    A = g.adj_parts[0].to_dense().double().cpu()
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = gcn.EpilogueGCNLayer.apply(*leaves, g.adj_parts, 'L2', act, skip)
    grads = torch.autograd.grad(y, leaves, dy)
    pre = (A @ x.double().cpu() @ w.double().cpu() + b.double().cpu()).requires_grad_(True)
    assert act != 'relu' or float(pre.abs().min()) > 1e-5
    a = _act(pre, act) * 1.0
    p, = torch.autograd.grad(a, pre, dy.double().cpu())
    ag = A @ p
    want = [a.detach() + (x.double().cpu() if skip else 0), ag @ w.double().cpu().t() + (dy.double().cpu() if skip else 0),
            x.double().cpu().t() @ ag, p.sum(0)]
    for got, ref, name in zip((y, *grads), want, ('y', 'dx', 'dw', 'db')):
        assert float((got.detach().double().cpu() - ref).abs().max()) <= 1e-5 * float(ref.abs().max()), name


def test_the_reference_model_on_fused_layers(env, golden_dir, monkeypatch):
    """DGNN_FUSED_LINEAR=1: the reference's loss curve, within the bar of the separate product and ReLU."""
    import dist_train
    w = np.load(os.path.join(golden_dir, 'tiny_P1.npz'))
    monkeypatch.setenv('DGNN_FUSED_LINEAR', '1')
    g = _graph(env, golden_dir, 'tiny')
    g.features = torch.from_numpy(w['r0_features']).to(env.device)
    assert dist_train.build_model(g, env).epilogue
    losses = dist_train.train(g, env, total_epoch=5)
    np.testing.assert_allclose(np.array(losses), w['r0_losses'], rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize('optimizer', ['adam', 'adamw', 'adamw8'])
def test_training_runs_and_repeats(env, golden_dir, optimizer):
    import dist_train
    runs = []
    for _ in range(2):
        g = _graph(env, golden_dir, 'ragged')
        runs.append(dist_train.train(g, env, total_epoch=4, hidden_dim=32, optimizer=optimizer, weight_decay=0.01, bias=True,
                                     activation='gelu', skip=True, eval_every=0))
    assert runs[0] == runs[1] and all(np.isfinite(runs[0])) and len(set(runs[0])) == 4
