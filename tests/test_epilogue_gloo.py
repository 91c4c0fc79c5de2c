"""Layers with bias, activation and skip connection in their product over 2 and 4 ranks (gloo, CPU): the layer against its
formulas on the unpartitioned graph in 64 bits, and two models that must not depend on the number of ranks. SpMM and layer
transform are swapped for CPU versions through the test hook."""
import os
import sys

import numpy as np
import pytest
import torch
import torch.multiprocessing as mp

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, 'tests'))
from test_variants_gloo import _cpu_gather, _free_port, _oracle_spmm, _raw  # noqa: E402

ACT = {'none': lambda t: t, 'relu': torch.relu, 'gelu': torch.nn.functional.gelu, 'silu': torch.nn.functional.silu}


class CpuDense:
    """spmm_cpp.linear's passes in plain torch; ``saved`` is x W + b."""

    @staticmethod
    def linear_forward(x, w, b=None, activation='none', residual=None, save=False):
        pre = x @ w if b is None else x @ w + b
        y = ACT[activation](pre)
        return (y if residual is None else y + residual), (pre if save else None)

    @staticmethod
    def linear_slope(dy, saved, activation, need_bias=True):
        with torch.enable_grad():
            t = saved.detach().requires_grad_(True)
            p, = torch.autograd.grad(ACT[activation](t) * 1.0, t, dy)
        return p, p.sum(0) if need_bias else None

    @staticmethod
    def linear_grad_input(p, w, add=None):
        return p @ w.t() if add is None else p @ w.t() + add

    @staticmethod
    def linear_grad_weight(x, p):
        return x.t() @ p


def scenario_layer(env, rank, world, gold_dir):
    import coo_graph
    from models import gcn
    gold = np.load(os.path.join(gold_dir, 'directed_graph.npz'))
    n = int(gold['num_nodes'])
    full = coo_graph.COO_Graph('directed', attr_dict=_raw(gold))
    parts = full.partition(world, save=False, with_transpose=True)
    A = torch.sparse_coo_tensor(torch.from_numpy(gold['adj_idx']), torch.from_numpy(gold['adj_val']), (n, n)).to_dense().double()
    out = {}
    for transposed in (False, True):
        g = coo_graph.Parted_COO_Graph('directed', rank, world, attr_dict=parts[rank], transposed_backward=transposed)
        s = g.local_num_nodes
        Ap = torch.zeros(s * world, s * world, dtype=torch.float64)
        Ap[:n, :n] = A
        back = Ap.t() if transposed else Ap                        # the reference aggregates with the same blocks (gcn.py:47)
        torch.manual_seed(7)
        X, W, b, G = torch.randn(s * world, 6), torch.randn(6, 6), torch.randn(6), torch.randn(s * world, 6)
        mine = slice(rank * s, (rank + 1) * s)
        for act in ACT:
            for skip in (False, True):
                x, w, c = X[mine].clone().requires_grad_(True), W.clone().requires_grad_(True), b.clone().requires_grad_(True)
                y = gcn.EpilogueGCNLayer.apply(x, w, c, g.adj_parts, 'L2', act, skip)
                y.backward(G[mine])
                pre = (Ap @ X.double() @ W.double() + b.double()).requires_grad_(True)
                a = ACT[act](pre)
                p, = torch.autograd.grad(a * 1.0, pre, G.double())
                ag = back @ p
                want = {'y': a.detach() + (X.double() if skip else 0), 'dx': ag @ W.double().t() + (G.double() if skip else 0)}
                err = {k: float((v[0].double() - v[1][mine]).abs().max() / v[1].abs().max())
                       for k, v in (('y', (y.detach(), want['y'])), ('dx', (x.grad, want['dx'])))}
                for k, got, ref in (('dw', w.grad, X.double().t() @ ag), ('db', c.grad, p.sum(0))):
                    err[k] = float((got.double() - ref).abs().max() / ref.abs().max())
                out[transposed, act, skip] = err
    os.environ['DGNN_WGRAD_FROM_Z'] = '1'
    x, w = X[mine].clone(), W.clone().requires_grad_(True)          # an input that needs no gradient: dW from the kept aggregation
    y = gcn.EpilogueGCNLayer.apply(x, w, None, g.adj_parts, 'L1', 'silu', False)
    y.backward(G[mine])
    pre = (Ap @ X.double() @ W.double()).requires_grad_(True)
    p, = torch.autograd.grad(ACT['silu'](pre), pre, G.double())
    ref = (Ap @ X.double()).t() @ p
    out['from_z'] = {'dw': float((w.grad.double() - ref).abs().max() / ref.abs().max())}
    try:
        gcn.EpilogueGCNLayer.apply(x, torch.randn(6, 4), None, g.adj_parts, 'L1', 'silu', True)
        out['square'] = {'refused': 1.0}
    except RuntimeError:
        out['square'] = {'refused': 0.0}
    return out


def scenario_models(env, rank, world, gold_dir):
    import coo_graph
    import dist_train
    gold = np.load(os.path.join(gold_dir, 'tiny_graph.npz'))
    full = coo_graph.COO_Graph('tiny', attr_dict=_raw(gold))
    out = {}
    for model, blocks, block in (('GCN', world, rank), ('GCN15D', world // 2, rank // 2)):
        if model == 'GCN15D' and world % 4:
            continue
        g = coo_graph.Parted_COO_Graph('tiny', block, blocks, attr_dict=full.partition(blocks, save=False)[block])
        net = dist_train.build_model(g, env, model, hidden_dim=8, num_layers=3, bias=True, activation='gelu', skip=True)
        with torch.no_grad():
            for p in net.parameters():
                p.sub_(0.4)
        opt = dist_train.build_optimizer(net.parameters(), 'adam')
        for _ in range(2):
            y, loss = dist_train.train_step(net, opt, lambda o, t: (torch.nn.functional.cross_entropy(o, t, reduction='sum') / 40), g, env)
        out[model] = {n: p.detach().double().numpy() for n, p in net.named_parameters()}
    return out


def _worker(rank, world, port, scenario, log_dir, q):
    try:
        for p in (ROOT, os.path.join(ROOT, 'dist-gnn_amd')):
            if p not in sys.path:
                sys.path.insert(0, p)
        torch.set_num_threads(1)
        os.environ.update(MASTER_ADDR='127.0.0.1', MASTER_PORT=str(port), DGNN_LOG_DIR=log_dir)
        import dist_utils
        from models import gcn
        gcn.set_spmm_backend(_oracle_spmm, gather=_cpu_gather, dense=CpuDense)
        env = dist_utils.DistEnv(rank, world, 'gloo', echo=False)
        q.put((rank, globals()['scenario_' + scenario](env, rank, world, os.path.join(ROOT, 'tests', 'golden'))))
        env.barrier_all()
        torch.distributed.destroy_process_group()
    except Exception:
        import traceback
        q.put((rank, {'error': traceback.format_exc()}))
        raise


def _run(world, scenario, tmp):
    ctx = mp.get_context('spawn')
    q = ctx.Queue()
    port = _free_port()
    procs = [ctx.Process(target=_worker, args=(r, world, port, scenario, tmp, q)) for r in range(world)]
    for p in procs:
        p.start()
    out = dict(q.get(timeout=240) for _ in range(world))
    for p in procs:
        p.join(timeout=60)
    for res in out.values():
        assert 'error' not in res, res.get('error')
    return out


def test_layer_matches_its_formulas_on_2_ranks(tmp_path):
    for res in _run(2, 'layer', str(tmp_path)).values():
        assert len(res) == 18
        for key, errs in res.items():
            assert all(e <= 1e-5 for e in errs.values()), (key, errs)


def test_models_do_not_depend_on_the_ranks(tmp_path):
    one, four = _run(1, 'models', str(tmp_path))[0]['GCN'], _run(4, 'models', str(tmp_path))
    assert 'bias3' in one and one['weight2'].shape == (8, 8)
    for res in four.values():
        for model in ('GCN', 'GCN15D'):
            for name, want in one.items():
                # two steps of 0.01: a gradient that is off by 1e-5 of its size moves a weight by 1e-7, one within rounding of
                # zero by whatever sign it has
                off = np.abs(res[model][name] - want)
                assert np.mean(off > 1e-5) < 0.02 and off.max() < 0.05, (model, name, off.max())


def test_options_are_checked():
    import dist_train
    with pytest.raises(ValueError, match='no bias'):
        dist_train.build_model(None, None, 'CachedGCN', bias=True)
    with pytest.raises(ValueError, match='no bias'):
        dist_train.build_model(None, None, 'AdaptiveGCN', activation='gelu')
    with pytest.raises(ValueError, match='unknown optimizer'):
        dist_train.build_optimizer([], 'sgd')
    with pytest.raises(ValueError, match='unknown activation'):
        dist_train.build_model(None, None, 'GCN', activation='tanh')
    import main
    args = main.parse_args(['--optimizer', 'adamw8', '--skip', '--bias', '--activation', 'gelu', '--weight-decay', '0.1'])
    assert args.optimizer == 'adamw8' and args.skip and args.bias and args.activation == 'gelu' and args.weight_decay == 0.1
    assert main.parse_args([]).optimizer == 'adam' and not main.parse_args([]).bias


def scenario_gradients(env, rank, world, gold_dir):
    import coo_graph
    import dist_train
    gold = np.load(os.path.join(gold_dir, 'tiny_graph.npz'))
    full = coo_graph.COO_Graph('tiny', attr_dict=_raw(gold))
    out = {}
    for model, blocks, block in (('GCN', world, rank), ('GCN15D', world // 2, rank // 2)):
        if model == 'GCN15D' and world % 4:
            continue
        g = coo_graph.Parted_COO_Graph('tiny', block, blocks, attr_dict=full.partition(blocks, save=False)[block])
        net = dist_train.build_model(g, env, model, hidden_dim=8, num_layers=3, bias=True, activation='gelu', skip=True)
        with torch.no_grad():
            for p in net.parameters():
                p.sub_(0.4)
        dist_train.train_step(net, torch.optim.SGD(net.parameters(), lr=0.01), lambda o, t: (torch.nn.functional.cross_entropy(o, t, reduction='sum') / 40), g, env)
        out[model] = {n: p.grad.double().numpy() for n, p in net.named_parameters()}
    return out


def test_gradients_do_not_depend_on_the_ranks(tmp_path):
    """The gradients themselves, before an optimiser makes steps of its own size of them: fp32 sums in another order, 1e-5 of the
    largest value."""
    one, four = _run(1, 'gradients', str(tmp_path))[0]['GCN'], _run(4, 'gradients', str(tmp_path))
    for res in four.values():
        assert set(res) == {'GCN', 'GCN15D'}
        for model in res:
            for name, want in one.items():
                assert np.abs(want).max() > 0
                assert np.abs(res[model][name] - want).max() <= 1e-5 * np.abs(want).max(), (model, name)
