"""The layer transform against its definition in 64 bits.

Bounds, with h = eps / 2 of the type (2^-24, bf16 2^-8, fp16 2^-11) and S = sum of |products|:
  sums        the fp32 accumulation of K products in 16s: at most (10 + 12 K / 16) 2^-24 S (six products an fp32 pair, each
              addition rounded once or truncated), a sixth of the K part for 16-bit operands; column sums are added in 64 bits: 4 2^-24 S
  result      h |result| on top
  activation  |act'| <= 1.13, |act''| <= 0.8; its own evaluation 16 2^-24 (|act| + |argument|)
  slope       x W + b is saved in fp32: 0.8 (2^-24 |pre| + its error) |dy|, and relu's bit may be either where |pre| is within
              its error; p is rounded once (h |p|) before the products
"""
import itertools

import numpy as np
import pytest
import torch

import spmm_cpp

pytestmark = pytest.mark.gpu

DT = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
HALF = {k: torch.finfo(t).eps / 2 for k, t in DT.items()}
U = 2.0 ** -24
SIZES = [(1, 1, 1), (4096, 3, 1), (1, 20, 4096), (63, 1433, 65), (64, 100, 65), (900, 5, 4), (3, 300, 4099), (8, 4100, 129), (4, 40, 8), (1, 602, 256), (2, 3, 5), (7, 4096, 130), (33, 17, 31), (31, 64, 32), (64, 1433, 16), (129, 40, 41), (257, 602, 256),
         (128, 256, 257), (300, 33, 300), (1000, 7, 64), (4099, 100, 47), (20000, 31, 129)]


def _inputs(m, k, n, dtype, bias, residual, seed, pad=0):
    gen = torch.Generator(device='cuda').manual_seed(seed)

    def t(*shape):
        wide = torch.full(shape[:-1] + (shape[-1] + pad,), float('nan'), device='cuda')          # what lies between rows is not a value
        wide[..., :shape[-1]] = torch.randn(*shape, generator=gen, device='cuda')
        return wide.to(DT[dtype])[..., :shape[-1]]
    x, w, dy = t(m, k), t(k, n), t(m, n)
    b = torch.randn(n, generator=gen, device='cuda').to(DT[dtype]) if bias else None
    return x, w, b, t(m, n) if residual else None, dy


def _d(t):
    return None if t is None else t.detach().double().cpu()


def _sum_bound(k, dtype):
    return (10 + (12 if dtype == 'f32' else 2) * k / 16) * U


def _act(a, act):
    if act == 'relu':
        return a.clamp_min(0), (a > 0).double()
    if act == 'gelu':
        cdf = 0.5 * torch.special.erfc(-a / 2 ** 0.5)
        return a * cdf, cdf + a * torch.exp(-a * a / 2) / (2 * np.pi) ** 0.5
    if act == 'silu':
        s = torch.sigmoid(a)
        return a * s, s * (1 + a * (1 - s))
    return a, torch.ones_like(a)


def _near(got, want, bound, name):
    off = (_d(got) - want).abs()
    assert got.shape == want.shape, name
    assert bool((off <= bound).all()), f'{name}: {float((off / bound.clamp_min(1e-300)).max()):.3g} times its bound'


def _definition(x, w, b, r, dy, dtype, act):
    """{name: (value, bound)} of the output and the gradients."""
    h, (x, w, b, r, dy) = HALF[dtype], map(_d, (x, w, b, r, dy))
    (m, k), n = x.shape, w.shape[1]
    pre, size = x @ w, x.abs() @ w.abs()
    if b is not None:
        pre, size = pre + b, size + b.abs()
    e_pre = _sum_bound(k, dtype) * size + U * pre.abs()
    y, slope = _act(pre, act)
    e_y = 1.13 * e_pre + 16 * U * (y.abs() + pre.abs())
    if r is not None:
        y = y + r
        e_y = e_y + U * y.abs()
    out = {'y': (y, e_y + h * y.abs() + 1e-40 + (2.0 ** -25 if dtype == 'f16' else 0))}
    p = dy * slope
    if act == 'none':
        e_p = torch.zeros_like(p)
    elif act == 'relu':
        e_p = dy.abs() * (pre.abs() <= e_pre)
    else:
        e_p = dy.abs() * (0.8 * (U * pre.abs() + 2 * e_pre) + 16 * U * (1 + pre.abs()))
    tiny = 2.0 ** -25 if dtype == 'f16' else 0               # fp16's smallest half step
    e_round = e_p + (h * (p.abs() + e_p) + tiny if act in ('gelu', 'silu') else 0)
    for name, a, c, e, count in (('dx', p, w.t(), None, n), ('dw', x.t(), p, None, m)):
        v = a @ c
        e = (e_round @ w.abs().t()) if name == 'dx' else (x.abs().t() @ e_round)
        e = e + _sum_bound(count, dtype) * (a.abs() @ c.abs() + e)
        out[name] = (v, e + h * v.abs() + 1e-40 + tiny)
    v = p.sum(0)
    e = e_p.sum(0) + 4 * U * (p.abs() + e_p).sum(0)
    out['db'] = (v, e + h * v.abs() + 1e-40 + tiny)
    out['dr'] = (dy, torch.zeros_like(dy))
    return out


def _run(x, w, b, r, dy, act):
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b, r) if t is not None]
    it = iter(leaves)
    xl, wl = next(it), next(it)
    bl = next(it) if b is not None else None
    rl = next(it) if r is not None else None
    y = spmm_cpp.linear(xl, wl, bl, activation=act, residual=rl)
    names = ['dx', 'dw'] + (['db'] if b is not None else []) + (['dr'] if r is not None else [])
    return {'y': y.detach(), **dict(zip(names, torch.autograd.grad(y, leaves, dy)))}


@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('m,k,n', SIZES)
def test_output_and_gradients(m, k, n, dtype):
    for i, act in enumerate(('none', 'relu', 'gelu', 'silu')):
        case = _inputs(m, k, n, dtype, i != 1, i >= 1, seed=m * 7 + n, pad=(0, 3, 8, 1)[i])
        want = _definition(*case, dtype, act)
        mine = _run(*case, act)
        for name, got in mine.items():
            assert got.dtype == DT[dtype]
            _near(got, *want[name], f'{act} {name}')
        assert torch.equal(spmm_cpp.linear(case[0], case[1], case[2], act, case[3]), mine['y'])      # saving nothing: the same bits


@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('m,k,n', [(65600, 70, 41), (65500, 130, 250), (33000, 520, 500)])
def test_output_and_gradients_of_many_rows(m, k, n, dtype):
    """Rows enough for weight gradients straight from memory and for two row blocks a wave, every side ragged."""
    for act, residual, pad in (('none', False, 0), ('gelu', True, 3)):
        case = _inputs(m, k, n, dtype, True, residual, seed=m + n, pad=pad)
        want = _definition(*case, dtype, act)
        mine = _run(*case, act)
        for name, got in mine.items():
            _near(got, *want[name], f'{act} {name}')
        assert torch.equal(spmm_cpp.linear(case[0], case[1], case[2], act, case[3]), mine['y'])


@pytest.mark.parametrize('dtype', list(DT))
def test_a_handful_of_rows(dtype):
    """1 to 9 rows against W as it lies and W^T, few and many columns: the crossover from multiply-adds to tiles on both sides."""
    for m, (k, n) in itertools.product((1, 2, 3, 4, 5, 8, 9), ((70, 41), (602, 256), (130, 4100), (2100, 1030))):
        case = _inputs(m, k, n, dtype, True, True, seed=m + n, pad=m % 2)
        want = _definition(*case, dtype, 'silu')
        for name, got in _run(*case, 'silu').items():
            _near(got, *want[name], f'{m}x{k}x{n} {name}')


@pytest.mark.parametrize('m,k,n', [(0, 5, 4), (3, 0, 4), (3, 5, 0), (0, 0, 0), (1, 0, 1)])
def test_empty_sides(m, k, n):
    for dtype, act in itertools.product(DT, ('none', 'relu', 'silu')):
        case = _inputs(m, k, n, dtype, True, True, seed=1)
        want = _definition(*case, dtype, act)
        for name, got in _run(*case, act).items():
            _near(got, *want[name], f'{act} {name}')


def test_fp32_is_as_exact_as_fp32_arithmetic():
    """The error against 64 bits is at most twice that of a plain chain of fp32 operations, over all outputs, for operands of
    ordinary size, of mixed sizes and with sums that cancel."""
    for seed, (m, k, n) in enumerate([(64, 8, 40), (64, 602, 64), (40, 4096, 300)]):
        x, w, _, _, _ = _inputs(m, k, n, 'f32', False, False, seed)
        for kind in ('plain', 'mixed', 'cancel'):
            if kind == 'mixed':
                x = x * torch.exp2(torch.randint(-20, 20, x.shape, device='cuda').float())
            if kind == 'cancel':
                x, w = torch.cat([x, x], 1), torch.cat([w, -w * (1 + 2.0 ** -10)], 0)
            want = _d(x) @ _d(w)
            xn, wn = x.cpu().numpy(), w.cpu().numpy()
            acc = np.zeros((m, n), np.float32)
            for i in range(x.shape[1]):
                acc += xn[:, i:i + 1] * wn[i]
            chain = float((torch.from_numpy(acc).double() - want).norm())
            mine = float((_d(spmm_cpp.linear(x, w)) - want).norm())
            assert mine <= 2 * chain, (kind, mine / chain)


def test_fp32_values_that_are_not_finite_or_near_the_edge():
    m, k, n = 70, 64, 80
    x, w, _, _, _ = _inputs(m, k, n, 'f32', False, False, 3)
    inf, big = float('inf'), 3.4e38
    x[3, 5], x[7, 1], x[9, 0], x[9, 1] = inf, -inf, inf, float('nan')
    x[12], w[:, 9] = 0, 0                                     # inf * 0 where row 3 meets column 9
    w[5, 11] = 0
    x[20] = 0
    x[20, 4] = big                                            # rounds to infinity in 8 bits
    w[:, 30] = 0
    w[4, 30] = 1.0
    w[2, 40] = inf
    for y, (a, b) in ((spmm_cpp.linear(x, w), (x, w)), (spmm_cpp.linear_grad_weight(x.t().contiguous(), w), (x, w)),
                      (spmm_cpp.linear_grad_input(x, w.t().contiguous()), (x, w))):
        want = (_d(a).unsqueeze(2) * _d(b).unsqueeze(0)).sum(1)        # the products as they are: inf * 0 is NaN
        want = want.float()                                            # and what passes fp32's range is infinity
        got = y.cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
        assert torch.equal(got[torch.isinf(got)], want[torch.isinf(want)])
        assert float(got[20, 30]) == float(torch.tensor(big))
        fine = torch.isfinite(want)
        assert torch.allclose(got[fine], want[fine], rtol=2e-5, atol=0.01)


@pytest.mark.parametrize('dtype', ['bf16', 'f16'])
def test_16_bit_values_that_are_not_finite(dtype):
    x, w, _, r, _ = _inputs(40, 64, 48, dtype, False, True, 4)
    x[3, 5], x[9, 1], r[11, 2] = float('inf'), float('nan'), float('nan')
    y = spmm_cpp.linear(x, w, None, 'relu', r)
    want = (_d(x).unsqueeze(2) * _d(w).unsqueeze(0)).sum(1)
    want = torch.where(want <= 0, torch.zeros_like(want), want) + _d(r)
    assert torch.equal(torch.isnan(y).cpu(), torch.isnan(want)) and torch.equal(torch.isinf(y).cpu(), torch.isinf(want))


def test_small_fp32_values():
    """Values of 2^-110 keep an absolute error of 2^-134 a unit of the other operand (bf16's smallest number is 2^-133)."""
    x, w, _, _, _ = _inputs(20, 40, 30, 'f32', False, False, 5)
    x = x * 2.0 ** -110
    want = _d(x) @ _d(w)
    bound = _sum_bound(40, 'f32') * (_d(x).abs() @ _d(w).abs()) + 3 * 2.0 ** -134 * _d(w).abs().sum(0)
    assert bool(((_d(spmm_cpp.linear(x, w)) - want).abs() <= bound).all())


def test_gradients_against_differences():
    """d loss along a random direction, from differences of the 64-bit definition at +-1e-6."""
    for act in ('gelu', 'silu', 'none'):
        x, w, b, r, dy = _inputs(37, 50, 45, 'f32', True, True, 6)
        g = _run(x, w, b, r, dy, act)
        gen = torch.Generator().manual_seed(1)
        for name, t in (('dx', x), ('dw', w), ('db', b), ('dr', r)):
            step = torch.randn(t.shape, generator=gen, dtype=torch.float64)

            def loss(e):
                args = [_d(x), _d(w), _d(b), _d(r)]
                args[('dx', 'dw', 'db', 'dr').index(name)] += e * step
                return float(((_act(args[0] @ args[1] + args[2], act)[0] + args[3]) * _d(dy)).sum())
            want = (loss(1e-6) - loss(-1e-6)) / 2e-6
            got = float((_d(g[name]) * step).sum())
            assert abs(got - want) <= 1e-4 * float((_d(g[name]).abs() * step.abs()).sum()), (act, name)


def test_only_what_is_asked_for():
    x, w, b, r, dy = _inputs(50, 20, 30, 'f32', True, True, 7)
    full = _run(x, w, b, r, dy, 'relu')
    for which in ('x', 'w', 'b', 'r'):
        ts = {'x': x.clone(), 'w': w.clone(), 'b': b.clone(), 'r': r.clone()}
        ts[which].requires_grad_(True)
        y = spmm_cpp.linear(ts['x'], ts['w'], ts['b'], 'relu', ts['r'])
        got, = torch.autograd.grad(y, ts[which], dy)
        assert torch.equal(got, full['d' + which])
    w = w.clone().requires_grad_(True)
    with pytest.raises(RuntimeError):                         # no second derivative
        g, = torch.autograd.grad(spmm_cpp.linear(x, w).sum(), w, create_graph=True)
        g.sum().backward()


def test_gradients_that_are_expanded_or_transposed():
    x, w, _, r, _ = _inputs(40, 24, 40, 'f32', False, True, 8)
    x.requires_grad_(True)
    y = spmm_cpp.linear(x, w, None, 'silu', r)
    a, = torch.autograd.grad(y.sum(), x)
    y = spmm_cpp.linear(x, w, None, 'silu', r)
    b, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(a, b)
    y = spmm_cpp.linear(x, w, None, 'silu', r)
    t = torch.randn(40, 40, device='cuda')
    c, = torch.autograd.grad(y.t(), x, t)
    y = spmm_cpp.linear(x, w, None, 'silu', r)
    d, = torch.autograd.grad(y, x, t.t().contiguous())
    assert torch.equal(c, d)


def test_a_skip_connections_gradient_joins_the_product():
    for dtype in DT:
        x, w, _, _, dy = _inputs(300, 70, 40, dtype, False, False, 15)
        want = _d(dy) @ _d(w).t() + _d(x)
        bound = _sum_bound(40, dtype) * (_d(dy).abs() @ _d(w).abs().t()) + (U + HALF[dtype]) * want.abs() + 2.0 ** -24
        _near(spmm_cpp.linear_grad_input(dy, w, add=x), want, bound, dtype)
    with pytest.raises(RuntimeError, match='add'):
        spmm_cpp.linear_grad_input(dy, w, add=x[:, :3])


def test_columns_between_rows_are_left_alone():
    """The C entries write rows of any distance and nothing between them."""
    x, w, b, r, dy = _inputs(100, 40, 70, 'f32', True, True, 9)
    y, saved = spmm_cpp.linear_forward(x, w, b, 'silu', r, save=True)
    p, db = spmm_cpp.linear_slope(dy, saved, 'silu')
    dx, dw = spmm_cpp.linear_grad_input(p, w), spmm_cpp.linear_grad_weight(x, p)
    lib, s = spmm_cpp.lib, spmm_cpp._stream(x)

    def room(m, n):
        return torch.full((m + 1, n + 5), 7.0, device='cuda')
    ws = torch.empty(1 << 22, device='cuda')
    Y, P, X, W = room(100, 70), room(100, 70), room(100, 40), room(40, 70)
    assert lib.dgnn_linear_forward(x.data_ptr(), 40, w.data_ptr(), 70, b.data_ptr(), r.data_ptr(), 70, Y.data_ptr(), 75, None, 0,
                                   100, 40, 70, 0, 3, ws.data_ptr(), ws.numel() * 4, s) == 0
    assert lib.dgnn_linear_slope(dy.data_ptr(), 70, saved.data_ptr(), 70, P.data_ptr(), 75, None, 100, 70, 0, 3, None, 0, s) == 0
    assert lib.dgnn_linear_grad_input(p.data_ptr(), 70, w.data_ptr(), 70, None, 0, X.data_ptr(), 45, 100, 40, 70, 0, ws.data_ptr(), ws.numel() * 4, s) == 0
    assert lib.dgnn_linear_grad_weight(x.data_ptr(), 40, p.data_ptr(), 70, W.data_ptr(), 75, 100, 40, 70, 0, ws.data_ptr(), ws.numel() * 4, s) == 0
    for big, small in ((Y, y), (P, p), (X, dx), (W, dw)):
        m, n = small.shape
        assert torch.equal(big[:m, :n], small)
        assert bool((big[m:] == 7).all()) and bool((big[:, n:] == 7).all())


def test_refusals_on_the_device():
    x, w, b, r, _ = _inputs(6, 4, 5, 'f32', True, True, 10)
    for kw in (dict(x=x.t()), dict(x=x.half()), dict(x=x.double()), dict(x=x[0]), dict(w=w.bfloat16()), dict(w=w[:3]), dict(b=b[:4]),
               dict(b=b.half()), dict(b=b.view(1, 5)), dict(r=r[:5]), dict(r=r[:1].expand(6, 5)), dict(act='tanh'), dict(act=None),
               dict(x=x[:1].expand(6, 4)), dict(w=w.cpu())):
        a = {**dict(x=x, w=w, b=b, r=r, act='relu'), **kw}
        with pytest.raises(RuntimeError, match='spmm_cpp.linear'):
            spmm_cpp.linear(a['x'], a['w'], a['b'], a['act'], a['r'])
    y, saved = spmm_cpp.linear_forward(x, w, b, 'gelu', r, save=True)
    for bad in (None, saved[:3], saved.half(), saved.t()):
        with pytest.raises(RuntimeError, match='saved'):
            spmm_cpp.linear_slope(y, bad, 'gelu')
    with pytest.raises(RuntimeError, match='shape'):
        spmm_cpp.linear_grad_weight(x, y[:5])
    with pytest.raises(RuntimeError, match='shape'):
        spmm_cpp.linear_grad_input(x, w)


@pytest.mark.parametrize('dtype,act,shape', [('f32', 'relu', (300, 602, 41)), ('bf16', 'gelu', (5, 600, 256)), ('f32', 'silu', (5000, 64, 64))])
def test_captured_and_replayed(dtype, act, shape):
    """Forward and backward captured twice, replayed with new inputs between eager work, the two graphs on two streams at once."""
    cases = [_inputs(*shape, dtype, True, True, seed) for seed in (11, 12)]
    graphs, outs = [], []
    leaves = [[t.clone().requires_grad_(True) for t in c[:4]] for c in cases]

    def work(l, dy):
        y = spmm_cpp.linear(l[0], l[1], l[2], act, l[3])
        return (y.detach(),) + torch.autograd.grad(y, l, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(leaves[0], cases[0][4])
    torch.cuda.current_stream().wait_stream(side)
    for l, c in zip(leaves, cases):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(work(l, c[4]))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(3):
        with torch.no_grad():
            for l in leaves:
                for t in l:
                    t.add_(0.25)
        want = [work(l, c[4]) for l, c in zip(leaves, cases)]
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                for _ in range(3):
                    g.replay()
        torch.cuda.synchronize()
        for o, e in zip(outs, want):
            for a, b in zip(o, e):
                assert torch.equal(a, b), turn


def test_two_streams_at_once():
    """Calls that cut their sums, on two streams: each has a workspace of its own."""
    cases = [_inputs(9, 4096, 200, 'f32', True, False, seed) for seed in (13, 14)]
    want = [spmm_cpp.linear(x, w, b, 'gelu') for x, w, b, _, _ in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                x, w, b, _, _ = cases[i]
                got[i].append(spmm_cpp.linear(x, w, b, 'gelu'))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, t) for t in g)


def test_offsets_past_32_bits():
    """Rows more than 2^32 bytes behind the first: 2^21 rows 1100 floats apart, the last ones checked."""
    m, k, n = 1 << 21, 40, 33
    buf = torch.zeros(m, 1100, device='cuda')
    x = buf[:, :k]
    gen = torch.Generator(device='cuda').manual_seed(0)
    tail = torch.randn(200, k, generator=gen, device='cuda')
    x[-200:] = tail
    w = torch.randn(k, n, generator=gen, device='cuda')
    y = spmm_cpp.linear(x, w)
    assert torch.equal(y[-200:], spmm_cpp.linear(tail, w)) and not bool(y[:-200].any())
    p = torch.zeros(m, n, device='cuda')
    p[-200:] = 1.0
    dw = spmm_cpp.linear_grad_weight(x, p)
    want = _d(tail).sum(0).unsqueeze(1).expand(k, n)
    assert bool(((_d(dw) - want).abs() <= _sum_bound(200, 'f32') * _d(tail).abs().sum(0).unsqueeze(1) + U * want.abs()).all())


def test_a_training_run_of_both_operators():
    """Layers and optimiser as they are used together: two layers, three steps, against the same in 64 bits. Each step moves a
    weight by at most about lr and gradients agree to 1e-5, so weights agree to 1e-4 lr; where a gradient is within rounding
    of zero its step's direction is noise, which is why weights with tiny gradients are left out."""
    gen = torch.Generator(device='cuda').manual_seed(3)
    x = torch.randn(500, 30, generator=gen, device='cuda')
    target = torch.randn(500, 6, generator=gen, device='cuda')
    shapes = [(30, 30), (30,), (30, 6), (6,)]
    ps = [torch.nn.Parameter(0.2 * torch.randn(*s, generator=gen, device='cuda')) for s in shapes]
    qs = [p.detach().double().cpu().requires_grad_(True) for p in ps]
    opt = spmm_cpp.AdamW(ps, lr=0.01, weight_decay=0.1, eps=1e-4)
    ref = torch.optim.AdamW(qs, lr=0.01, weight_decay=0.1, eps=1e-4)
    xd, td = x.double().cpu(), target.double().cpu()
    for _ in range(3):
        h = spmm_cpp.linear(x, ps[0], ps[1], 'gelu', residual=x)
        y = spmm_cpp.linear(h, ps[2], ps[3])
        loss = (y - target).square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        hd = torch.nn.functional.gelu(xd @ qs[0] + qs[1]) + xd
        ld = (hd @ qs[2] + qs[3] - td).square().mean()
        ref.zero_grad()
        ld.backward()
        ref.step()
        assert abs(float(loss) - float(ld)) < 1e-5 * float(ld)
    for p, q in zip(ps, qs):
        # a step is lr g / (|g| + eps)-like: its slope in g is at most lr / eps = 100, gradients are off by < 1e-7
        assert float((p.double().cpu() - q).abs().max()) < 3 * 100 * 1e-7 + 1e-6


@pytest.mark.parametrize('m', [40, 3000])
def test_operands_that_share_a_buffer_by_columns(m):
    """x, y, what is saved, dx and dy in columns of one buffer, the bias gradient between two of its rows: nothing overlaps, and
    the results are those of separate matrices. An input gradient over x itself is refused with nothing written."""
    k, n = 40, 70
    x, w, b, r, dy = _inputs(m, k, n, 'f32', True, False, 21)
    y, saved = spmm_cpp.linear_forward(x, w, b, 'gelu', None, save=True)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    dx, dw, db = torch.autograd.grad(spmm_cpp.linear(*leaves, 'gelu'), leaves, dy)
    lib, s, f = spmm_cpp.lib, spmm_cpp._stream(x), 4
    pitch = k + 3 * n + k + n                                  # x | y | saved | dy | dx | room for db in a row
    buf = torch.full((m, pitch), 7.0, device='cuda')
    at = [buf.data_ptr() + f * o for o in (0, k, k + n, k + 2 * n, k + 3 * n, k + 3 * n + k)]
    buf[:, :k], buf[:, k + 2 * n:k + 3 * n] = x, dy
    ws = torch.empty(1 << 23, device='cuda')
    assert lib.dgnn_linear_forward(at[0], pitch, w.data_ptr(), n, b.data_ptr(), None, 0, at[1], pitch, at[2], pitch, m, k, n, 0, 2, ws.data_ptr(), ws.numel() * 4, s) == 0
    dw2 = torch.empty(k, n, device='cuda')
    before = buf.clone()
    assert lib.dgnn_linear_backward(at[0], pitch, w.data_ptr(), n, at[3], pitch, at[2], pitch, at[0], pitch, dw2.data_ptr(), n, at[5], m, k, n, 0, 2, ws.data_ptr(),
                                    ws.numel() * 4, s) == 1
    assert torch.equal(buf, before)
    assert lib.dgnn_linear_backward(at[0], pitch, w.data_ptr(), n, at[3], pitch, at[2], pitch, at[4], pitch, dw2.data_ptr(), n, at[5], m, k, n, 0, 2, ws.data_ptr(),
                                    ws.numel() * 4, s) == 0
    parts = buf.split([k, n, n, n, k, n], 1)
    for got, want in zip(parts, (x, y, saved, dy, dx)):
        assert torch.equal(got, want)
    assert torch.equal(parts[5][0], db) and bool((parts[5][1:] == 7).all()) and torch.equal(dw2, dw)


def test_derivatives_that_would_be_dropped_are_refused():
    """Forward mode on each operand, forward over backward, a trace, and function transforms: none returns a value without its
    derivative."""
    x, w, b, r, dy = _inputs(6, 4, 5, 'f32', True, True, 22)
    for at in range(4):
        for grad in (False, True):
            with torch.autograd.forward_ad.dual_level():
                ops = [t.clone().requires_grad_(grad) for t in (x, w, b, r)]
                ops[at] = torch.autograd.forward_ad.make_dual(ops[at], torch.ones_like(ops[at]))
                with pytest.raises(RuntimeError, match='forward-mode|forward mode'):
                    spmm_cpp.linear(ops[0], ops[1], ops[2], 'gelu', ops[3])
    xl = x.clone().requires_grad_(True)
    y = spmm_cpp.linear(xl, w, b, 'gelu', r)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match='forward-mode'):
            torch.autograd.grad(y, xl, torch.autograd.forward_ad.make_dual(dy, torch.ones_like(dy)))
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: spmm_cpp.linear(t, w, b, 'gelu', r), (x,), (torch.ones_like(x),))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: spmm_cpp.linear(t, w, b, 'gelu', r).sum())(x)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: spmm_cpp.linear(t, w, b, 'gelu', r))(x.expand(3, 6, 4))
    with pytest.raises(RuntimeError, match='torch.jit.trace'):
        torch.jit.trace(lambda t: spmm_cpp.linear(t, w, b, 'gelu', r), x, check_trace=False)


def test_a_gradient_that_is_stored_negated():
    """The gradient of a column that became the imaginary part of a conjugate comes back as a view with its sign set lazily."""
    x, w, b, _, _ = _inputs(50, 4, 1, 'f32', True, False, 23)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = spmm_cpp.linear(*leaves, 'silu')
    dy = torch._neg_view(torch.randn(50, 1, device='cuda'))
    assert dy.is_neg()
    got = torch.autograd.grad(y, leaves, dy)
    want = torch.autograd.grad(spmm_cpp.linear(*leaves, 'silu'), leaves, dy.resolve_neg())
    assert all(torch.equal(a, c) for a, c in zip(got, want))


def _ieee(a, b):
    """a b in 64 bits with every product of a row or column that is not finite as IEEE has it (inf * 0 is NaN), and the bound of
    its finite values' fp32 sums."""
    fa, fb = (torch.where(torch.isfinite(t), t, torch.zeros_like(t)) for t in (a, b))
    out = fa @ fb
    for i in torch.nonzero(~torch.isfinite(a).all(1)).view(-1).tolist():
        out[i] = (a[i].unsqueeze(1) * b).sum(0)
    for j in torch.nonzero(~torch.isfinite(b).all(0)).view(-1).tolist():
        out[:, j] = (a * b[:, j]).sum(1)
    return out, _sum_bound(a.shape[1], 'f32') * (fa.abs() @ fb.abs())


def _like_ieee(got, clean, a, b, bias=None):
    """Infinities and NaN are fp32's own, finite values hold their bound, rows and columns without such values (if there are some) the very bits
    they have when there are none anywhere."""
    a, b = _d(a), _d(b)
    want, bound = _ieee(a, b)
    if bias is not None:
        want, bound = want + _d(bias), bound + U * _d(bias).abs()
    want = want.float()                                       # past fp32's range is infinity
    got, clean = got.cpu(), clean.cpu()
    # where an infinity stands in a sum whose finite terms alone can pass fp32's range (bound / bound's factor is their absolute
    # sum), a part of the sum can be an infinity of the other sign: which of infinity and NaN it gives is the order of the parts
    both = torch.isinf(want) & (bound > 3.4e38 * _sum_bound(a.shape[1], 'f32')) & ~(torch.isfinite(a).all(1).unsqueeze(1) & torch.isfinite(b).all(0).unsqueeze(0))
    assert not bool(torch.isfinite(got[both]).any())
    got, want = got.masked_fill(both, 0), want.masked_fill(both, 0)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
    assert torch.equal(got[torch.isinf(got)], want[torch.isinf(want)])
    fine = torch.isfinite(want)
    assert bool(((got.double() - want.double()).abs() <= bound + 2 * U * want.double().abs())[fine].all())
    same = (torch.isfinite(a) & (a.abs() < 1e30)).all(1).unsqueeze(1) & (torch.isfinite(b) & (b.abs() < 1e30)).all(0).unsqueeze(0)
    assert torch.equal(got[same], clean[same])


@pytest.mark.parametrize('m,k,n', [(4227, 203, 70), (4230, 130, 300), (12300, 70, 41), (16500, 9, 20), (300, 500, 50), (70, 64, 80)])
def test_fp32_values_that_are_not_finite_at_many_sizes(m, k, n):
    """Rows enough for the kernels that take rows straight from memory, W as it lies and W^T, every side ragged, NaN between the
    rows; and the tiles' kernels, cut along the contraction or not."""
    inf, nan, big = float('inf'), float('nan'), 3.4e38
    x, w, b, _, p = _inputs(m, k, n, 'f32', True, False, 31, pad=3)

    def mild(t):
        return torch.where(t.abs() < 1e30, t, torch.zeros_like(t))

    def spoil(t):
        t = t.clone()
        r, c = t.shape
        t[3, 5], t[33, 1], t[r - 1, 0], t[40, 2], t[40, 7] = inf, -inf, nan, inf, -inf
        t[64 % r, c - 1] = big                                # rounds to infinity in 8 bits
        t[50, :] = 0
        return t
    xs, ps, ws = spoil(x), spoil(p), w.clone()
    ws[:, 6] = 0                                              # inf * 0
    ws[:, 8] = 0
    ws[4, 8], ws[2, 9 % n], ws[k - 1, n - 1] = 100.0, inf, -big
    for c in (w, ws):
        _like_ieee(spmm_cpp.linear(xs, c, b), spmm_cpp.linear(mild(xs), mild(c), b), xs, c, b)
    _like_ieee(spmm_cpp.linear_grad_input(ps, w), spmm_cpp.linear_grad_input(mild(ps), w), ps, w.t())
    one = xs[:, 8:9]
    _like_ieee(spmm_cpp.linear_grad_weight(one, p), spmm_cpp.linear_grad_weight(mild(one), p), one.t(), p)


@pytest.mark.parametrize('m,k,n', [(65600, 70, 41), (65700, 140, 20), (66000, 33, 100)])
def test_fp32_weight_gradients_of_many_rows_that_are_not_finite(m, k, n):
    inf = float('inf')
    x, _, _, _, p = _inputs(m, k, n, 'f32', False, False, 32, pad=1)
    xs, ps = x.clone(), p.clone()
    xs[70, 3], xs[40000, 3], xs[m - 1, 7], xs[12, 11], xs[5, 20], xs[9, 32] = inf, inf, -inf, float('nan'), 3.4e38, 3.0e38
    ps[70, :] = ps[70, :].abs() + 1
    ps[40000, :] = ps[40000, :].abs() + 1
    ps[40000, 5] = -1.0                                       # inf - inf where row 70 and this one meet
    ps[m - 1, 9] = 0.0                                        # inf * 0
    ps[9, :] *= 100                                           # past fp32's range
    ps[33, 15] = inf
    mild = [torch.where(t.abs() < 1e30, t, torch.zeros_like(t)) for t in (xs, ps)]
    _like_ieee(spmm_cpp.linear_grad_weight(xs, ps), spmm_cpp.linear_grad_weight(*mild), xs.t(), ps)


def test_infinity_times_the_smallest_numbers():
    """An infinity times a number below the normal ones is an infinity."""
    for m in (70, 4230):
        x, w, _, _, _ = _inputs(m, 130, 70, 'f32', False, False, 33)
        x[5, 3], w[3, :] = float('inf'), 1e-40
        w[3, 1] = -1e-42
        y = spmm_cpp.linear(x, w)[5]
        assert float(y[1]) == -float('inf') and bool((torch.cat([y[:1], y[2:]]) == float('inf')).all())


@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('m,k,n', [(4096, 1024, 1), (1024, 2050, 3), (4096, 250, 1), (2048, 500, 1), (1000, 2048, 4), (2049, 33, 1), (128, 70, 16), (129, 70, 16), (3, 600, 700)])
def test_gradients_of_tall_narrow_layers(m, k, n, dtype):
    """On both sides of the rule for backward passes in one launch."""
    for act, pad in (('gelu', 0), ('relu', 3), ('none', 1)):
        case = _inputs(m, k, n, dtype, True, act == 'relu', seed=m + k, pad=pad)
        want = _definition(*case, dtype, act)
        for name, got in _run(*case, act).items():
            _near(got, *want[name], f'{act} {name}')


@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('m,k,n', [(4227, 203, 70), (12300, 40, 256), (33000, 520, 130), (65600, 16, 97)])
def test_relu_over_several_words_of_saved_bits(m, k, n, dtype):
    """Rows enough for the kernel that takes them straight from memory, more columns than one word, ragged or not."""
    case = _inputs(m, k, n, dtype, True, n == 256, seed=41, pad=3)
    want = _definition(*case, dtype, 'relu')
    for name, got in _run(*case, 'relu').items():
        _near(got, *want[name], f'relu {name}')


@pytest.mark.parametrize('dtype', ['bf16', 'f16'])
@pytest.mark.parametrize('m,k,n', [(1, 602, 256), (8, 100, 64), (64, 1433, 16), (33, 40, 31), (1024, 64, 2), (5, 3, 4)])
def test_small_16_bit_layers_round_their_gradients_once(m, k, n, dtype):
    """A backward pass in one launch keeps p = dy act'(x W + b) in fp32 (sizes of small_fit): its gradients carry their own
    rounding and what fp32 arithmetic loses, not p's 16 bits."""
    for act in ('gelu', 'silu'):
        x, w, b, _, dy = case = _inputs(m, k, n, dtype, True, False, seed=42)
        got = _run(*case, act)
        h, tiny = HALF[dtype], 2.0 ** -25 if dtype == 'f16' else 0
        x, w, b, dy = map(_d, (x, w, b, dy))
        pre, size = x @ w + b, x.abs() @ w.abs() + b.abs()
        e_pre = _sum_bound(k, dtype) * size + U * pre.abs()
        p = dy * _act(pre, act)[1]
        # act's 16-bit evaluation: a tail of 1e-6 relative error and the operations around it, within 32 U of the slope's terms
        e_p = dy.abs() * (0.8 * (U * pre.abs() + 2 * e_pre) + 32 * U * (1 + pre.abs()))
        for name, a, c, e, count in (('dx', p, w.t(), e_p @ w.abs().t(), n), ('dw', x.t(), p, x.abs().t() @ e_p, m)):
            v = a @ c
            _near(got[name], v, e + _sum_bound(count, 'f32') * (a.abs() @ c.abs() + e) + h * v.abs() + 1e-40 + tiny, f'{act} {name}')


@pytest.mark.parametrize('dtype', ['bf16', 'f16'])
@pytest.mark.parametrize('m,k,n', [(3000, 20, 3), (6030, 3054, 1), (2200, 1, 88), (700, 33, 64), (700, 33, 65), (20000, 602, 41), (65600, 3, 5), (9, 2, 1973), (33, 5000, 63), (500, 63, 65)])
def test_narrow_16_bit_layers_round_their_weight_gradients_once(m, k, n, dtype):
    """dw of layers of few columns, or of few weights, carries its own rounding, what fp32 sums lose and the rounding of p's second
    16-bit piece, not that of p = dy act'(x W + b) itself. x positive, as behind an activation, so that nothing averages."""
    for act, pad in (('gelu', 0), ('silu', 3)):
        x, w, b, _, dy = case = _inputs(m, k, n, dtype, True, False, seed=51, pad=pad)
        x.abs_()
        got = _run(*case, act)
        h, tiny = HALF[dtype], 2.0 ** -25 if dtype == 'f16' else 0
        x, w, b, dy = map(_d, (x, w, b, dy))
        pre, size = x @ w + b, x.abs() @ w.abs() + b.abs()
        e_pre = _sum_bound(k, dtype) * size + U * pre.abs()
        p = dy * _act(pre, act)[1]
        e_p = dy.abs() * (0.8 * (U * pre.abs() + 2 * e_pre) + 32 * U * (1 + pre.abs()))
        e_p = e_p + h * h * (p.abs() + e_p) + tiny
        v, e = x.t() @ p, x.abs().t() @ e_p
        _near(got['dw'], v, (e + _sum_bound(m, dtype) * 2 * (x.abs().t() @ p.abs() + e)) * (1 + h) + h * v.abs() + 1e-40 + tiny, f'{act} dw')


@pytest.mark.parametrize('dtype', ['bf16', 'f16'])
def test_narrow_16_bit_weight_gradients_that_are_not_finite(dtype):
    """An infinity times p is an infinity of its sign, whatever p's two pieces are; NaN stays where it is."""
    m, k, n = 4000, 12, 9
    x, w, b, _, dy = _inputs(m, k, n, dtype, True, False, 52)
    x.mul_(0.25)
    w[3], w[5], w[7] = 0, 0, 0                                # so that x W + b stays finite
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = spmm_cpp.linear(*leaves, 'gelu')
    clean = torch.autograd.grad(y, leaves[1], dy, retain_graph=True)[0]
    inf = float('inf')
    with torch.no_grad():
        leaves[0].data[10, 3], leaves[0].data[20, 5], leaves[0].data[30, 5], leaves[0].data[40, 7] = inf, inf, -inf, float('nan')
    got = torch.autograd.grad(y, leaves[1], dy)[0]
    pre = _d(x) @ _d(w) + _d(b)
    p = _d(dy) * _act(pre, 'gelu')[1]
    assert bool((p[[10, 20, 30]].abs() > 1e-3).any())
    want = torch.zeros(k, n, dtype=torch.float64)
    want[3] = inf * p[10]
    want[5] = inf * p[20] - inf * p[30]
    want[7] = float('nan')
    for row in (3, 5, 7):
        g = got[row].cpu()
        assert torch.equal(torch.isnan(g), torch.isnan(want[row])) and torch.equal(g[torch.isinf(g)].double(), want[row][torch.isinf(want[row])])
    rest = [i for i in range(k) if i not in (3, 5, 7)]
    assert torch.equal(got[rest], clean[rest])


@pytest.mark.parametrize('dtype', ['bf16', 'f16'])
@pytest.mark.parametrize('m,k,n', [(9, 2, 1973), (1, 46, 4251), (45, 1, 47), (77, 23, 300), (1, 2048, 2100), (2048, 1, 3), (2, 1024, 1030), (2, 1025, 1030)])
def test_input_gradients_of_few_values_round_once(m, k, n, dtype):
    """dx of at most 2048 values carries its own rounding and what fp32 sums lose; beyond, the rounding of p too."""
    for act, pad in (('gelu', 3), ('silu', 0)):
        x, w, b, _, dy = case = _inputs(m, k, n, dtype, True, False, seed=61, pad=pad)
        w.abs_()
        got = _run(*case, act)
        h, tiny = HALF[dtype], 2.0 ** -25 if dtype == 'f16' else 0
        x, w, b, dy = map(_d, (x, w, b, dy))
        pre, size = x @ w + b, x.abs() @ w.abs() + b.abs()
        e_pre = _sum_bound(k, dtype) * size + U * pre.abs()
        p = dy * _act(pre, act)[1]
        e_p = dy.abs() * (0.8 * (U * pre.abs() + 2 * e_pre) + 32 * U * (1 + pre.abs()))
        if m * k > 2048:
            e_p = e_p + h * (p.abs() + e_p) + tiny
        v, e = p @ w.t(), e_p @ w.abs().t()
        _near(got['dx'], v, (e + _sum_bound(n, 'f32') * (p.abs() @ w.abs().t() + e)) * (1 + h) + h * v.abs() + 1e-40 + tiny, f'{act} dx')


@pytest.mark.parametrize('dtype,act,shape', [('bf16', 'gelu', (40, 30, 64)), ('f16', 'silu', (3000, 20, 41)), ('f32', 'gelu', (4230, 130, 70))])
def test_captured_and_replayed_on_other_kernels(dtype, act, shape):
    """Weight gradients from two pieces of p, input gradients of few values, rows straight from memory."""
    test_captured_and_replayed(dtype, act, shape)
