"""AdamW on the GPU against numpy: in 64 bits (the definition) and, for the 8-bit codes, in 32 bits in the header's order of
operations (every operation there is rounded once, so codes and scales must agree to the bit)."""
import copy

import numpy as np
import pytest
import torch

import spmm_cpp

pytestmark = pytest.mark.gpu

LR, B1, B2, EPS, DECAY = 0.01, 0.9, 0.999, 1e-8, 0.01
DT = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
SIZES = (1, 3, 255, 256, 257, 4095, 4096, 4097, 70001)


def _params(sizes, dtype, seed, gap=0):
    """Parameters cut out of one buffer, `gap` elements apart (so most start at odd places), and gradients of three sizes."""
    gen = torch.Generator(device='cuda').manual_seed(seed)
    buf = torch.randn(sum(sizes) + gap * len(sizes) + 1, generator=gen, device='cuda').mul_(0.05).to(dtype)
    out, at = [], gap
    for k, n in enumerate(sizes):
        p = torch.nn.Parameter(buf[at:at + n])
        out.append(p)
        at += n + gap
    return out


def _grads(params, seed):
    gen = torch.Generator(device='cuda').manual_seed(1000 + seed)
    for k, p in enumerate(params):
        p.grad = (torch.randn(p.shape, generator=gen, device='cuda') * (10.0 ** -(k % 3))).to(p.dtype)


def _np(t):
    return t.detach().float().cpu().numpy()


def _codes_np(x, root, t, along, ahead):
    """Header's rounding in float32: (values of the codes, scales)."""
    n, f = x.size, np.float32
    pad = np.zeros(-(-n // 256) * 256, f)
    pad[:n] = x
    pad = pad.reshape(-1, 256)
    top = np.maximum(np.abs(pad).max(1, keepdims=True), f(2.0 ** -100))
    c = pad * (f(448) / top)
    e = np.maximum(np.frexp(c)[1] - 1, -6)
    s = np.ldexp(f(1), e - 3).astype(f)
    i = np.arange(pad.size, dtype=np.uint64)
    h = (i * np.uint64(along) + np.uint64(t) * np.uint64(ahead)) & np.uint64(0xFFFFFFFF)
    u = ((h >> np.uint64(16)).astype(f) * f(2.0 ** -16)).reshape(pad.shape)
    q = np.copysign(np.floor(np.abs(c) / s + u) * s, c).astype(f)
    if root:
        q = np.where((pad > 0) & (q < f(2.0 ** -9)), f(2.0 ** -9), q)
    return q.reshape(-1)[:n], (top * f(f(1) / f(448))).reshape(-1)


class _Twin:
    """The header's step in float32 (bit for bit) or float64."""

    def __init__(self, p, bits, master, f):
        self.p, self.bits, self.master, self.f, self.t = _np(p).astype(f), bits, master, f, 0
        z = np.zeros_like(self.p)
        self.m, self.v, self.codes = z.copy(), z.copy(), None

    def step(self, g, dtype, lr=LR, decay=DECAY):
        f = self.f
        self.t += 1
        g = g.astype(f)
        self.m = self.m * f(B1) + g * f(1 - B1)
        self.v = self.v * f(B2) + (g * g) * f(1 - B2)
        r = np.sqrt(self.v)
        step = self.m / (r * f(1 / np.sqrt(1 - B2 ** self.t)) + f(EPS))
        p = self.p * f(1 - lr * decay) - step * f(lr / (1 - B1 ** self.t))
        self.wide = p
        self.p = p if self.master or dtype == torch.float32 else _np(torch.from_numpy(p.astype(np.float32)).to(dtype)).astype(f)
        if self.bits == 8:
            mq, ms = _codes_np(self.m.astype(np.float32), False, self.t, 0x6A09E667, 0x9E3779B9)
            rq, rs = _codes_np(r.astype(np.float32), True, self.t, 0x3C6EF372, 0xBB67AE85)
            self.codes = mq, ms, rq, rs
            n = mq.size
            self.m = (mq * np.repeat(ms, 256)[:n]).astype(f)
            self.v = np.square((rq * np.repeat(rs, 256)[:n]).astype(f))


def _check_state(opt, p, twin, dtype, exact):
    st = opt.state[p]
    assert int(st['step']) == twin.t
    if opt.state_bits == 8:
        mq, ms, rq, rs = twin.codes
        for name, want in (('exp_avg', mq), ('exp_avg_scale', ms), ('exp_avg_rms', rq), ('exp_avg_rms_scale', rs)):
            assert np.array_equal(_np(st[name]).reshape(-1), want), name
    elif exact:
        assert np.array_equal(_np(st['exp_avg']).reshape(-1), twin.m) and np.array_equal(_np(st['exp_avg_sq']).reshape(-1), twin.v)
    if exact:
        if opt.master_weights:
            assert np.array_equal(_np(st['master']).reshape(-1), twin.wide)
        want = _np(torch.from_numpy(twin.wide).to(dtype))
        assert np.array_equal(_np(p).reshape(-1), want)


CASES = [('f32', False), ('bf16', False), ('f16', False), ('bf16', True), ('f16', True)]


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('dtype,master', CASES)
def test_steps_to_the_bit(dtype, master, bits):
    params = _params(SIZES, DT[dtype], 1, gap=3)
    buf = params[0]._base if params[0]._base is not None else None
    opt = spmm_cpp.AdamW(params, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=DECAY, state_bits=bits, master_weights=master)
    twins = [_Twin(p, bits, master, np.float32) for p in params]
    for k in range(3):
        _grads(params, k)
        opt.step()
        for p, t in zip(params, twins):
            t.step(_np(p.grad).reshape(-1), DT[dtype])
            _check_state(opt, p, t, DT[dtype], True)
    del buf


@pytest.mark.parametrize('dtype,master', CASES)
def test_codes_over_the_whole_range(dtype, master):
    """Blocks of gradients that fit one another and blocks whose values lie many powers of ten apart, are zero but for one in
    ten, or whose squares are below the normal numbers: the same bits, whichever way a wave rounds and takes its roots."""
    params = _params((256 * 40 + 37, 256 * 8), DT[dtype], 11)
    opt = spmm_cpp.AdamW(params, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=DECAY, state_bits=8, master_weights=master)
    twins = [_Twin(p, 8, master, np.float32) for p in params]
    rng = np.random.default_rng(5)
    for k in range(3):
        for p, t in zip(params, twins):
            n = p.numel()
            g, block = rng.standard_normal(n), np.arange(n) // 256
            kind = (block + 3 * k) % 5
            g = np.where(kind == 1, g * 10.0 ** rng.uniform(-12, 2, n), g)
            g = np.where((kind == 2) & (rng.random(n) < 0.9), 0.0, g)
            g = np.where(kind == 3, g * 1e-22, g)
            g = np.where((kind == 4) & (block % 2 == 0), 0.0, g)
            p.grad = torch.from_numpy(g.astype(np.float32)).cuda().to(p.dtype)
        opt.step()
        for p, t in zip(params, twins):
            t.step(_np(p.grad).reshape(-1), DT[dtype])
            _check_state(opt, p, t, DT[dtype], True)


def test_against_64_bits():
    """fp32 moments and parameters after 5 steps within what their roundings allow: m and v lose at most 3 half steps a step
    (two products, a sum), the update 6 more relative to itself, the parameter 2 relative to itself."""
    params = _params(SIZES, torch.float32, 2)
    opt = spmm_cpp.AdamW(params, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=DECAY)
    twins = [_Twin(p, 32, False, np.float64) for p in params]
    half = 2.0 ** -24
    slack = [np.zeros_like(t.p) for t in twins]
    for k in range(5):
        _grads(params, k)
        opt.step()
        for t, p, s in zip(twins, params, slack):
            before = t.p.copy()
            t.step(_np(p.grad).reshape(-1), torch.float32)
            # |m / denom| in these steps is at most 4; m's terms may cancel: its error is relative to the terms' sizes, at most
            # 3 half steps a step of (sum of |terms|) <= 4 * 0.32 denom-sized values -> 24 half steps of the rate in all
            s += 3 * half * np.abs(before) + LR / (1 - B1 ** t.t) * 4 * (6 + 15 + 15) * half
    for t, p, s in zip(twins, params, slack):
        assert np.all(np.abs(_np(p).reshape(-1) - t.p) <= s)
        assert np.allclose(_np(opt.state[p]['exp_avg_sq']).reshape(-1), t.v, rtol=15 * half, atol=0)


def test_neighbours_of_a_tensor_are_left_alone():
    buf = torch.full((5000,), 7.0, device='cuda', dtype=torch.bfloat16)
    p = torch.nn.Parameter(buf[1001:1001 + 2111])
    p.grad = torch.ones_like(p)
    spmm_cpp.AdamW([p], lr=1.0, state_bits=8).step()           # 7 has steps of 1/32 in bf16
    assert bool((buf[:1001] == 7).all()) and bool((buf[3112:] == 7).all()) and bool((p != 7).any())


def test_many_tensors_one_call():
    """More tensors than one launch takes, empty ones and ones without a gradient among them."""
    sizes = [int(n) for n in np.random.RandomState(0).randint(0, 900, 150)]
    params = _params(sizes, torch.float32, 3)
    _grads(params, 0)
    idle = list(range(5, 150, 11))
    for i in idle:
        params[i].grad = None
    before = [p.detach().clone() for p in params]
    opt = spmm_cpp.AdamW(params, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=DECAY)
    twins = [_Twin(p, 32, False, np.float32) for p in params]
    opt.step()
    for i, (p, t) in enumerate(zip(params, twins)):
        if i in idle:
            assert torch.equal(p, before[i]) and int(opt.state[p]['step']) == 0
        else:
            t.step(_np(p.grad).reshape(-1), torch.float32)
            _check_state(opt, p, t, torch.float32, True)
    _grads(params, 1)                                       # now step counts differ from tensor to tensor
    for i, (p, t) in enumerate(zip(params, twins)):
        t.step(_np(p.grad).reshape(-1), torch.float32)
    opt.step()
    for p, t in zip(params, twins):
        _check_state(opt, p, t, torch.float32, True)


def test_groups_schedules_and_strided_gradients():
    a, b = _params((300, 520), torch.float32, 4)
    w = torch.nn.Parameter(torch.randn(20, 30, device='cuda'))
    opt = spmm_cpp.AdamW([{'params': [a], 'lr': 0.1, 'weight_decay': 0.0}, {'params': [b, w]}], lr=LR, betas=(B1, B2), eps=EPS, weight_decay=DECAY)
    sched = torch.optim.lr_scheduler.LambdaLR(opt, lambda t: 1.0 / (1 + t))
    twins = [_Twin(p.reshape(-1), 32, False, np.float32) for p in (a, b, w)]
    for k in range(2):
        _grads([a, b], k)
        w.grad = torch.randn(30, 20, device='cuda').t()     # not contiguous
        opt.step()
        for p, t, lr, wd in zip((a, b, w), twins, (0.1 / (1 + k), LR / (1 + k), LR / (1 + k)), (0.0, DECAY, DECAY)):
            t.step(_np(p.grad).reshape(-1), torch.float32, lr, wd)
            assert np.array_equal(_np(p).reshape(-1), t.p)
        sched.step()
    late = torch.nn.Parameter(torch.ones(77, device='cuda'))
    opt.add_param_group({'params': [late]})
    late.grad = torch.ones_like(late)
    opt.step()
    assert int(opt.state[late]['step']) == 1 and int(opt.state[a]['step']) == 3 and bool((late < 1).all())


@pytest.mark.parametrize('bits,master', [(32, False), (8, False), (8, True)])
def test_state_dict_and_copies_continue(bits, master, tmp_path):
    dtype = torch.bfloat16 if master else torch.float32
    params = _params((257, 1000), dtype, 5)
    opt = spmm_cpp.AdamW(params, state_bits=bits, master_weights=master)
    _grads(params, 0)
    opt.step()
    torch.save(opt.state_dict(), tmp_path / 'opt.pt')
    saved = torch.load(tmp_path / 'opt.pt', weights_only=True)
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    other = spmm_cpp.AdamW(twins, state_bits=bits, master_weights=master)
    other.load_state_dict(saved)
    both = copy.deepcopy((params, opt))
    for k in (1, 2):
        _grads(params, k)
        for t, c, p in zip(twins, both[0], params):
            t.grad, c.grad = p.grad.clone(), p.grad.clone()
        opt.step()
        other.step()
        both[1].step()
    for p, t, c in zip(params, twins, both[0]):
        assert torch.equal(p, t) and torch.equal(p, c)
        for name in opt.state[p]:
            if name != 'step':
                assert torch.equal(opt.state[p][name].float(), other.state[t][name].float()), name
    flat = opt.state_buffers()
    assert flat['exp_avg'].numel() == 512 + 1024 and flat['exp_avg'].data_ptr() == opt.state[params[0]]['exp_avg'].data_ptr()
    with pytest.raises(ValueError, match='does not fit'):
        spmm_cpp.AdamW(twins, state_bits=40 - bits).load_state_dict(saved)


def test_master_follows_a_parameter_that_somebody_wrote():
    p = torch.nn.Parameter(torch.randn(600, device='cuda').bfloat16())
    opt = spmm_cpp.AdamW([p], lr=LR, master_weights=True)
    p.grad = torch.randn_like(p)
    opt.step()
    with torch.no_grad():
        p.copy_(torch.full_like(p, 3.0))
    p.grad = torch.zeros_like(p)
    opt.step()
    assert bool((opt.state[p]['master'] > 2.8).all()) and bool((opt.state[p]['master'] < 3.2).all())
    p.data[:300] = -1.0                                      # no version counter sees this
    kept = opt.state[p]['master'][300:].clone()
    opt.step()
    assert bool((opt.state[p]['master'][:300] < -0.9).all())
    step = (opt.state[p]['master'][300:] - kept).abs()
    assert bool((step < LR).all()) and bool((opt.state[p]['master'][300:] != p[300:].float()).any())


def test_autograd_notices_the_write():
    w = torch.nn.Parameter(torch.randn(8, device='cuda'))
    opt = spmm_cpp.AdamW([w])
    y = (w * w).sum()
    w.grad = torch.ones_like(w)
    opt.step()
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.backward()


def test_refusals_on_the_device():
    p = torch.nn.Parameter(torch.randn(64, device='cuda'))
    for bad in ([torch.nn.Parameter(torch.randn(8, 8, device='cuda').t())], [torch.nn.Parameter(torch.randn(8, device='cuda').double())],
                [torch.nn.Parameter(p.detach()[:40]), torch.nn.Parameter(p.detach()[30:])]):
        with pytest.raises(RuntimeError, match='AdamW'):
            spmm_cpp.AdamW(bad)
    with pytest.raises(RuntimeError, match='master_weights'):
        spmm_cpp.AdamW([p], master_weights=True)
    opt = spmm_cpp.AdamW([p])
    p.grad = torch.zeros(64, device='cuda').to_sparse()
    with pytest.raises(RuntimeError, match='gradient'):
        opt.step()
    assert int(opt.state[p]['step']) == 0


@pytest.mark.parametrize('bits', [32, 8])
def test_values_that_are_not_finite_stay_in_their_block(bits):
    p = torch.nn.Parameter(torch.ones(1000, device='cuda'))
    opt = spmm_cpp.AdamW([p], state_bits=bits)
    for k in range(3):
        p.grad = torch.full_like(p, 0.5)
        if k == 0:
            p.grad[300], p.grad[301] = float('nan'), float('inf')
        opt.step()
    bad = ~torch.isfinite(p.detach())
    want = torch.zeros_like(bad)
    if bits == 32:
        want[300:302] = True
    else:
        want[256:512] = True
    assert torch.equal(bad, want)


def test_codes_follow_a_slow_average():
    """With gradients whose size drops to a third in half of a block's elements the 8-bit second moment has to follow there
    (rounded to nearest it would stay within a code of where it was, 9 times too high). Over 3000 steps the average's memory
    of the old size is exp(-3); the mean over 2000 elements of stored / true varies by its 35 % scatter / sqrt(2000) < 1 %,
    and a root that scatters by 17 % squares to a mean 3 % high: within 15 %."""
    n = 4096
    gen = torch.Generator(device='cuda').manual_seed(0)
    p = torch.nn.Parameter(torch.zeros(n, device='cuda'))
    opt = spmm_cpp.AdamW([p], lr=0.0, state_bits=8)
    size = torch.ones(n, device='cuda')
    true = torch.zeros(n, device='cuda', dtype=torch.float64)
    for t in range(4000):
        if t == 1000:
            size[::2] /= 3
        p.grad = torch.randn(n, generator=gen, device='cuda') * size
        true.mul_(0.999).add_(p.grad.double().square(), alpha=0.001)
        opt.step()
    st = opt.state[p]
    v = (st['exp_avg_rms'].float().view(-1, 256) * st['exp_avg_rms_scale'].unsqueeze(1)).square().view(-1).double()
    for half in (slice(0, None, 2), slice(1, None, 2)):
        assert abs(float((v[half] / true[half]).mean()) - 1) < 0.15


@pytest.mark.parametrize('bits,dtype,master', [(32, 'f32', False), (8, 'bf16', True)])
def test_captured_steps(bits, dtype, master):
    """A captured step replayed with new gradients between eager work gives the eager optimiser's bits."""
    mine, theirs = _params((500, 4097, 3), DT[dtype], 6), None
    theirs = [torch.nn.Parameter(p.detach().clone()) for p in mine]
    kw = dict(lr=LR, betas=(B1, B2), eps=EPS, weight_decay=DECAY, state_bits=bits, master_weights=master)
    opt, eager = spmm_cpp.AdamW(mine, capturable=True, **kw), spmm_cpp.AdamW(theirs, **kw)
    fixed = [torch.zeros_like(p) for p in mine]
    for p, g in zip(mine, fixed):
        p.grad = g
    _grads(theirs, 9)
    eager.init_state()
    with pytest.raises(RuntimeError, match='capturable=True'):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            eager.step()
    with pytest.raises(RuntimeError, match='before capturing'):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    opt.init_state()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for k in range(4):
        _grads(theirs, k)
        for g, p in zip(fixed, theirs):
            g.copy_(p.grad)
        graph.replay()
        torch.cuda.synchronize()
        eager.step()
        torch.randn(1000, device='cuda').sum().item()
        for p, q in zip(mine, theirs):
            assert torch.equal(p, q), k
            assert int(opt.state[p]['step']) == int(eager.state[q]['step']) == k + 1


def test_another_stream():
    params = _params((100000, 50), torch.float32, 7)
    twins = [_Twin(p, 32, False, np.float32) for p in params]
    opt = spmm_cpp.AdamW(params, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=DECAY)
    s = torch.cuda.Stream()
    _grads(params, 0)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        opt.step()
    torch.cuda.current_stream().wait_stream(s)
    for p, t in zip(params, twins):
        t.step(_np(p.grad).reshape(-1), torch.float32)
        _check_state(opt, p, t, torch.float32, True)


def test_element_numbers_past_32_bits():
    """A tensor of more than 2^31 bytes and a state that starts past it: byte offsets that do not fit 32 bits."""
    n = (1 << 31) + 4096 + 77
    p = torch.nn.Parameter(torch.ones(n, device='cuda', dtype=torch.bfloat16))
    q = torch.nn.Parameter(torch.ones(300, device='cuda', dtype=torch.bfloat16))
    opt = spmm_cpp.AdamW([p, q], lr=0.5, weight_decay=0.0, state_bits=8)
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    opt.step()
    assert bool((p == 0.5).all()) and bool((q == 0.5).all())
    del opt, p, q
    torch.cuda.empty_cache()



def test_more_chunks_than_one_side_of_a_grid():
    """2^33 elements are 2^23 workgroups and some, more than a grid takes along one side."""
    if torch.cuda.mem_get_info()[0] < 120 << 30:
        pytest.skip('needs 120 GB of device memory')
    n = (1 << 33) + 5000
    p = torch.nn.Parameter(torch.ones(n, device='cuda', dtype=torch.bfloat16))
    opt = spmm_cpp.AdamW([p], lr=0.5, weight_decay=0.0, state_bits=8, master_weights=True)
    p.grad = torch.ones_like(p)
    opt.step()
    assert bool((p == 0.5).all())
    del opt, p
    torch.cuda.empty_cache()


def test_a_gradient_that_is_stored_negated():
    p, q = (torch.nn.Parameter(torch.ones(300, device='cuda')) for _ in range(2))
    g = torch.randn(300, device='cuda')
    p.grad, q.grad = torch._neg_view(g), -g
    assert p.grad.is_neg()
    spmm_cpp.AdamW([p, q]).step()
    assert torch.equal(p, q)


@pytest.mark.parametrize('bits,dtype,master', [(32, 'f32', False), (8, 'bf16', True)])
def test_a_state_loaded_behind_a_captured_step(bits, dtype, master):
    """A checkpoint is loaded into the buffers that a captured step writes: its replays go on from the loaded state, as an eager
    optimiser that loads the same does."""
    kw = dict(lr=LR, betas=(B1, B2), eps=EPS, weight_decay=DECAY, state_bits=bits, master_weights=master)
    mine = _params((500, 4097, 3), DT[dtype], 16)
    theirs = [torch.nn.Parameter(p.detach().clone()) for p in mine]
    opt, eager = spmm_cpp.AdamW(mine, capturable=True, **kw), spmm_cpp.AdamW(theirs, **kw)
    for k in range(2):
        _grads(theirs, k)
        for p, q in zip(mine, theirs):
            p.grad = q.grad.clone()
        opt.step()
        eager.step()
    saved = copy.deepcopy(opt.state_dict())
    start = [p.detach().clone() for p in mine]
    places = {n: t.data_ptr() for n, t in opt.state_buffers().items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    graph.replay()
    opt.load_state_dict(saved)
    eager.load_state_dict(saved)
    assert places == {n: t.data_ptr() for n, t in opt.state_buffers().items()}
    with torch.no_grad():
        for p, q, s in zip(mine, theirs, start):
            p.copy_(s)
            q.copy_(s)
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(mine, theirs):
            q.grad = p.grad.clone()
        eager.step()
        for p, q in zip(mine, theirs):
            assert torch.equal(p, q) and int(opt.state[p]['step']) == int(eager.state[q]['step']) == k + 3
            for n, x in opt.state[p].items():
                assert n == 'step' or torch.equal(x.float(), eager.state[q][n].float()), n


def test_a_state_that_does_not_fit_changes_nothing():
    params = _params((300, 700), torch.float32, 17)
    opt = spmm_cpp.AdamW(params, lr=LR)
    _grads(params, 0)
    opt.step()
    good = copy.deepcopy(opt.state_dict())
    before = {n: t.clone() for n, t in opt.state_buffers().items()}
    short, odd, less = copy.deepcopy(good), copy.deepcopy(good), copy.deepcopy(good)
    short['state'][1]['exp_avg_sq'] = short['state'][1]['exp_avg_sq'][:-1]
    del odd['state'][1]['exp_avg']
    less['param_groups'][0]['params'] = [0]
    for bad in (short, odd, less):
        with pytest.raises(ValueError):
            opt.load_state_dict(bad)
        assert all(torch.equal(t, before[n]) for n, t in opt.state_buffers().items()) and int(opt.state[params[1]]['step']) == 1
        assert opt.state[params[0]]['exp_avg'].data_ptr() == opt.state_buffers()['exp_avg'].data_ptr()
    opt.step()
    assert int(opt.state[params[0]]['step']) == 2


def test_loading_permuted_partial_and_hooked_states():
    """Two parameters' own states exchanged, one left out, and hooks that change what is loaded and see what was."""
    params = _params((300, 300), torch.float32, 18)
    opt = spmm_cpp.AdamW(params, lr=LR)
    _grads(params, 0)
    opt.step()
    a, b = (opt.state[p]['exp_avg'].clone() for p in params)
    given = opt.state_dict()
    opt.load_state_dict({**given, 'state': {0: given['state'][1], 1: given['state'][0]}})
    assert torch.equal(opt.state[params[0]]['exp_avg'], b) and torch.equal(opt.state[params[1]]['exp_avg'], a)
    given = copy.deepcopy(opt.state_dict())
    opt.load_state_dict({**given, 'state': {0: given['state'][0]}})
    assert torch.equal(opt.state[params[0]]['exp_avg'], b) and not opt.state[params[1]]['exp_avg'].any() and int(opt.state[params[1]]['step']) == 0
    seen = []
    opt.register_load_state_dict_pre_hook(lambda o, d: {**d, 'state': {i: {**s, 'step': 40 + i} for i, s in d['state'].items()}})
    opt.register_load_state_dict_post_hook(lambda o: seen.append([int(o.state[p]['step']) for p in params]))
    opt.load_state_dict(given)
    assert seen == [[40, 41]]


def test_parameters_that_left_their_group():
    """The optimiser steps what param_groups holds, never a tensor that was replaced there; late additions get their state."""
    a, b, c = (torch.nn.Parameter(torch.ones(n, device='cuda')) for n in (300, 20, 300))
    opt = spmm_cpp.AdamW([a, b], lr=LR)
    for p in (a, b, c):
        p.grad = torch.ones_like(p)
    opt.step()
    kept = [p.detach().clone() for p in (a, b, c)]
    group = opt.param_groups[0]
    for params in ([c, b], [a], [a, c]):
        group['params'] = params
        with pytest.raises(RuntimeError, match='replaced'):
            opt.step()
        assert all(torch.equal(p, k) for p, k in zip((a, b, c), kept))
    cpu = torch.nn.Parameter(torch.ones(3))
    cpu.grad = torch.ones(3)
    for params, why in (([a, b, cpu], 'no CPU path'), ([a, b, a], 'twice'), ([a, b, torch.nn.Parameter(a.detach()[5:9])], 'overlap')):
        group['params'] = params
        with pytest.raises(RuntimeError, match=why):
            opt.step()
    for params in ([b, a], [b, c, a]):
        group['params'] = params
        opt.step()
    assert [int(opt.state[p]['step']) for p in (a, b, c)] == [3, 3, 1]
    other = spmm_cpp.AdamW([c, b], lr=LR)
    other.load_state_dict({'state': {1: opt.state_dict()['state'][0]}, 'param_groups': [{**other.state_dict()['param_groups'][0]}]})
    assert int(other.state[b]['step']) == 3
    group['params'] = [a, b, c]
    opt.step()
    opt.param_groups.append({**group, 'params': [torch.nn.Parameter(torch.ones(3, device='cuda'))]})
    opt.init_state()
    del opt.param_groups[1]
    with pytest.raises(RuntimeError, match='replaced'):
        opt.step()


def test_a_step_that_is_refused_steps_nothing():
    """Whatever is wrong with a later group, the earlier ones stay as they are, and the next step is their first."""
    a, b, c = (torch.nn.Parameter(torch.ones(n, device='cuda', dtype=t)) for n, t in ((300, torch.float32), (20, torch.bfloat16), (30, torch.float32)))
    opt = spmm_cpp.AdamW([{'params': [a, b]}, {'params': [c]}], lr=LR)
    for p in (a, b, c):
        p.grad = torch.ones_like(p)
    good, last = c.grad, opt.param_groups[1]
    c.grad = good.to_sparse()
    with pytest.raises(RuntimeError, match='gradient'):
        opt.step()
    c.grad = good
    for name, x in (('lr', float('nan')), ('weight_decay', -1.0), ('weight_decay', float('nan')), ('eps', float('inf')), ('betas', (0.9, 1.0))):
        kept = last[name]
        last[name] = x
        with pytest.raises(ValueError, match='AdamW'):
            opt.step()
        last[name] = kept
    torch.cuda.synchronize()
    assert all(bool((p == 1).all()) and int(opt.state[p]['step']) == 0 for p in (a, b, c))
    opt.step()
    assert all(bool((p < 1).all()) and int(opt.state[p]['step']) == 1 for p in (a, b, c))


def test_a_group_that_is_refused_is_not_there():
    a, b = (torch.nn.Parameter(torch.ones(n, device='cuda')) for n in (300, 20))
    opt = spmm_cpp.AdamW([a], lr=LR)
    for bad in ({'params': [b], 'lr': -1.0}, {'params': [b], 'weight_decay': float('nan')}, {'params': [b], 'betas': (0.9,)},
                {'params': [b, torch.nn.Parameter(a.detach()[3:9])]}, {'params': [torch.nn.Parameter(torch.ones(3))]}):
        with pytest.raises((RuntimeError, ValueError), match='AdamW'):
            opt.add_param_group(bad)
        assert len(opt.param_groups) == 1
    opt.add_param_group({'params': [b], 'lr': 0.0})
    a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
    opt.step()
    assert bool((a < 1).all()) and len(opt.param_groups) == 2 and int(opt.state[b]['step']) == 1


def test_a_given_state_survives_a_refusal():
    """A state that a copy brought along is still there after a first step that was refused for another parameter."""
    a, b = _params((300, 20), torch.float32, 19)
    first = spmm_cpp.AdamW([a, b], lr=LR)
    _grads([a, b], 0)
    first.step()
    opt = spmm_cpp.AdamW([a, b], lr=LR)
    for p in (a, b):
        opt.state[p] = {n: x.clone() for n, x in first.state[p].items()}
    group = opt.param_groups[0]
    group['params'] = [a, b, torch.nn.Parameter(torch.ones(3))]
    with pytest.raises(RuntimeError, match='no CPU path'):
        opt.step()
    group['params'] = [a, b]
    opt.state[b]['exp_avg'] = opt.state[b]['exp_avg'][:-1]
    with pytest.raises(ValueError, match='size'):
        opt.step()
    opt.state[b]['exp_avg'] = first.state[b]['exp_avg'].clone()
    opt.step()
    first.param_groups[0]['lr'] = 0.0
    first.step()
    for p in (a, b):
        assert int(opt.state[p]['step']) == 2 and torch.equal(opt.state[p]['exp_avg'], first.state[p]['exp_avg'])
