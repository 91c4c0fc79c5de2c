"""The layer transform's refusals: its C entries' checks (nothing is launched) and the binding's."""
import ctypes

import pytest
import torch

import spmm_cpp

A, B, C, D = 1 << 22, 2 << 22, 3 << 22, 4 << 22             # addresses nobody reads: every call here is refused before a launch
lib = spmm_cpp.lib


def _forward(x=A, ldx=8, w=B, ldw=8, bias=None, res=None, ldr=0, y=C, ldy=8, save=None, lds=0, M=4, K=8, N=8, dtype=0, act=0, ws=None, n=0):
    return lib.dgnn_linear_forward(x, ldx, w, ldw, bias, res, ldr, y, ldy, save, lds, M, K, N, dtype, act, ws, n, None)


def _slope(dy=A, ldd=8, save=B, lds=8, p=C, ldp=8, db=None, M=4, N=8, dtype=0, act=2, ws=None, n=0):
    return lib.dgnn_linear_slope(dy, ldd, save, lds, p, ldp, db, M, N, dtype, act, ws, n, None)


def _grad_input(p=A, ldp=8, w=B, ldw=8, add=None, lda=8, dx=C, ldx=8, M=4, K=8, N=8, dtype=0, ws=None, n=0):
    return lib.dgnn_linear_grad_input(p, ldp, w, ldw, add, lda, dx, ldx, M, K, N, dtype, ws, n, None)


def _grad_weight(x=A, ldx=8, p=B, ldp=8, dw=C, ldw=8, M=4, K=8, N=8, dtype=0, ws=None, n=0):
    return lib.dgnn_linear_grad_weight(x, ldx, p, ldp, dw, ldw, M, K, N, dtype, ws, n, None)


def _backward(x=A, ldx=8, w=B, ldw=8, dy=C, ldd=8, save=D, lds=8, dx=5 << 22, lddx=8, dw=6 << 22, lddw=8, db=7 << 22, M=4, K=8, N=8, dtype=0, act=2,
              ws=8 << 22, n=1 << 20):
    return lib.dgnn_linear_backward(x, ldx, w, ldw, dy, ldd, save, lds, dx, lddx, dw, lddw, db, M, K, N, dtype, act, ws, n, None)


@pytest.mark.parametrize('call,kw', [
    (_forward, dict(dtype=3)), (_forward, dict(act=4)), (_forward, dict(act=-1)), (_forward, dict(M=-1)), (_forward, dict(K=1 << 31)),
    (_forward, dict(x=None)), (_forward, dict(w=None)), (_forward, dict(y=None)), (_forward, dict(ldx=7)), (_forward, dict(ldw=7)),
    (_forward, dict(ldy=7)), (_forward, dict(x=A + 2)), (_forward, dict(bias=A + 1)), (_forward, dict(res=D, ldr=7)),
    (_forward, dict(y=A + 64)), (_forward, dict(y=B)), (_forward, dict(res=C + 32, ldr=8)), (_forward, dict(act=1, save=D, lds=0)),
    (_forward, dict(act=2, save=D, lds=7)), (_forward, dict(M=9, K=4096, N=64, ldx=4096, ldw=64, ldy=64, x=1 << 30)),      # cut, no workspace
    (_slope, dict(dtype=-1)), (_slope, dict(act=9)), (_slope, dict(save=None)), (_slope, dict(lds=7)), (_slope, dict(dy=None)),
    (_slope, dict(ldp=7)), (_slope, dict(act=1, lds=0)), (_slope, dict(db=D)), (_slope, dict(db=D, ws=D, n=4)), (_slope, dict(db=D + 2)),
    (_grad_input, dict(dtype=5)), (_grad_input, dict(p=None)), (_grad_input, dict(ldx=7)), (_grad_input, dict(dx=A)), (_grad_input, dict(add=D, lda=7)), (_grad_input, dict(add=C)), (_grad_input, dict(N=-2)),
    (_backward, dict(dtype=5)), (_backward, dict(act=4)), (_backward, dict(M=-1)), (_backward, dict(M=600, ws=None)), (_backward, dict(M=600, n=100)),
    (_backward, dict(M=600, ws=(8 << 22) + 8)), (_backward, dict(ldx=7)), (_backward, dict(w=None)), (_backward, dict(M=600, dy=None)), (_backward, dict(lddw=3)),
    (_backward, dict(db=(7 << 22) + 2)), (_backward, dict(dx=B)), (_backward, dict(dw=C)), (_backward, dict(act=1, lds=0)), (_backward, dict(dy=None)), (_backward, dict(save=None)),
    (_grad_weight, dict(dtype=5)), (_grad_weight, dict(x=None)), (_grad_weight, dict(ldw=7)), (_grad_weight, dict(dw=B)),
    (_grad_weight, dict(M=1 << 31)), (_grad_weight, dict(M=100000, dw=1 << 40)),                                # cut, no workspace
])
def test_c_entries_refuse(call, kw):
    assert call(**kw) == 1 and b'linear' in lib.dgnn_last_error()


@pytest.mark.parametrize('call,kw', [
    (_forward, dict(K=(1 << 24) + 1)), (_forward, dict(N=(1 << 24) + 1)), (_grad_weight, dict(K=(1 << 24) + 1)), (_slope, dict(N=(1 << 24) + 1)),
    (_forward, dict(M=(1 << 31) - 1, y=1 << 44, w=1 << 50)), (_grad_input, dict(M=(1 << 31) - 1, dx=1 << 44, w=1 << 50)),          # 2^24 tiles
    (_grad_weight, dict(M=64, K=1 << 24, N=1 << 15, ldx=1 << 24, ldp=1 << 15, ldw=1 << 15, dw=1 << 50)),
])
def test_c_entries_refuse_what_a_launch_cannot_hold(call, kw):
    assert call(**kw) == 1 and b'linear' in lib.dgnn_last_error()


def test_c_entries_with_nothing_to_do():
    assert _forward(M=0, x=None, y=None) == 0 and _forward(N=0, w=None, y=None) == 0 and _grad_input(M=0, p=None, dx=None) == 0
    assert _grad_weight(K=0, x=None, dw=None) == 0 and _slope(N=0, dy=None, save=None, p=None) == 0 and _slope(M=0, dy=None, save=None, p=None) == 0


def test_workspace_is_bounded():
    """Only products with fewer tiles than compute units are cut, so the partial sums stay under 256 tiles of 128 x 256 floats;
    where W is laid out, its image has at most 6 bytes an element, both sides rounded up (to 256 and 64); the weight gradient's
    partial sums weigh at most a quarter of its operands, and one output at least."""
    n = ctypes.c_int64()
    for kind in range(4):
        for M in (0, 1, 7, 33, 2708, 232965, 2449029):
            for K in (0, 1, 100, 602, 4096):
                for N in (0, 1, 16, 41, 256, 4096):
                    for dtype in range(3):
                        assert lib.dgnn_linear_workspace(kind, M, K, N, dtype, ctypes.byref(n)) == 0
                        assert 0 <= n.value <= (max(256 * 128 * 256 * 4, 6 * (K + 256) * (N + 256), M * (K + N), 4 * K * N) if kind != 1 else 4096 * max(N, 1) * 8)
    assert lib.dgnn_linear_workspace(4, 1, 1, 1, 0, ctypes.byref(n)) == 1
    assert lib.dgnn_linear_workspace(0, -1, 1, 1, 0, ctypes.byref(n)) == 1
    assert lib.dgnn_linear_workspace(0, 1, 1, 1, 0, None) == 1


def test_binding_refuses_cpu_tensors_and_other_things():
    x, w = torch.zeros(3, 4), torch.zeros(4, 5)
    with pytest.raises(RuntimeError, match='no CPU path'):
        spmm_cpp.linear(x, w)
    with pytest.raises(RuntimeError, match='no CPU path'):
        spmm_cpp.linear(x.requires_grad_(True), w)
    with pytest.raises(RuntimeError, match='must be a torch.Tensor'):
        spmm_cpp.linear([[1.0]], w)
    for f in (spmm_cpp.linear_grad_input, spmm_cpp.linear_grad_weight):
        with pytest.raises(RuntimeError, match='no CPU path'):
            f(x, w)
    with pytest.raises(RuntimeError, match='no CPU path'):
        spmm_cpp.linear_slope(x.detach(), None, 'none')


# 4 x 8 x 8 takes one launch, 600 x 8 x 8 a launch for each gradient; dx, dw, db, x, w, dy and what was saved all lie apart in _backward
@pytest.mark.parametrize('M', [4, 600])
@pytest.mark.parametrize('kw', [
    dict(dx=A), dict(dx=A + 32), dict(dx=B), dict(dx=C), dict(dx=D), dict(dw=A), dict(dw=C + 96), dict(dw=D + 64), dict(db=A + 32), dict(db=B + 32),
    dict(db=C), dict(db=D + 32), dict(dx=5 << 22, dw=5 << 22), dict(dx=5 << 22, db=(5 << 22) + 64), dict(dw=6 << 22, db=(6 << 22) + 32),
    dict(dx=A, dw=None, w=A), dict(dw=B, dx=None, x=B),
])
def test_backward_refuses_outputs_that_overlap(M, kw):
    """Before any launch, whichever way the sizes take: an input gradient over x would be read as x by x^T p."""
    assert _backward(M=M, **kw) == 1 and b'overlap' in lib.dgnn_last_error()


def test_backward_refuses_before_it_launches():
    """Sizes that the last product of the call cannot launch, with every operand in order."""
    big = dict(M=1 << 13, K=1 << 24, N=1 << 15, ldx=1 << 24, ldw=1 << 15, ldd=1 << 15, lds=1 << 15, lddx=1 << 24, lddw=1 << 15, act=0, x=1 << 50, w=2 << 50, dy=3 << 50,
               dx=4 << 50, dw=5 << 50, db=6 << 50, n=1 << 60)
    assert _backward(**big) == 1 and b'tiles' in lib.dgnn_last_error()


@pytest.mark.parametrize('call,kw', [
    (_forward, dict(save=C, lds=8, act=2)), (_forward, dict(save=A, lds=8, act=3)), (_forward, dict(save=B + 32, lds=1, act=1)), (_forward, dict(bias=C + 32)),
    (_forward, dict(res=D, ldr=8, save=D, lds=8, act=2)), (_slope, dict(p=A + 32)), (_slope, dict(p=A, ldp=16)), (_slope, dict(p=B)), (_slope, dict(db=A, ws=D, n=1 << 20)),
    (_slope, dict(db=B + 32, ws=D, n=1 << 20)), (_slope, dict(db=C, ws=D, n=1 << 20)), (_slope, dict(p=A, db=A + 32, ws=D, n=1 << 20)),
])
def test_passes_refuse_operands_that_overlap(call, kw):
    assert call(**kw) == 1 and b'overlap' in lib.dgnn_last_error()


def _passes():
    x, w, b, r = torch.zeros(3, 4), torch.zeros(4, 5), torch.zeros(5), torch.zeros(3, 5)
    return {'linear': (spmm_cpp.linear, [x, w, b, 'none', r]), 'linear_forward': (spmm_cpp.linear_forward, [x, w, b, 'relu', r, True]),
            'linear_slope': (spmm_cpp.linear_slope, [r, r, 'silu']), 'linear_grad_input': (spmm_cpp.linear_grad_input, [r, w, x]),
            'linear_grad_weight': (spmm_cpp.linear_grad_weight, [x, r])}


@pytest.mark.parametrize('name', ['linear', 'linear_forward', 'linear_slope', 'linear_grad_input', 'linear_grad_weight'])
def test_forward_mode_derivatives_are_refused(name):
    """A dual tensor's tangent would be dropped, and its derivative read as zero. Refused before the device is looked at."""
    f, args = _passes()[name]
    with torch.autograd.forward_ad.dual_level():
        args[0] = torch.autograd.forward_ad.make_dual(args[0], torch.ones_like(args[0]))
        with pytest.raises(RuntimeError, match='forward-mode'):
            f(*args)


@pytest.mark.parametrize('name', ['linear', 'linear_forward', 'linear_slope', 'linear_grad_input', 'linear_grad_weight'])
def test_tracing_is_refused(name):
    """A trace would record the empty output alone and replay whatever its memory holds."""
    f, args = _passes()[name]
    first, rest = args[0], args[1:]
    with pytest.raises(RuntimeError, match='torch.jit.trace'):
        torch.jit.trace(lambda t: f(t, *rest), first, check_trace=False)


def test_values_that_are_stored_negated_are_refused():
    """One column of a conjugate's imaginary part is a plain float column by its strides; its memory holds the values' negatives."""
    z = torch.complex(torch.ones(3, 1), torch.ones(3, 1)).conj().imag
    assert z.is_neg()
    with pytest.raises(RuntimeError, match='resolve_neg'):
        spmm_cpp.linear(z, torch.zeros(1, 5))


def test_small_backward_passes_are_bounded_by_what_they_repeat():
    """A backward pass without workspace is the one that runs in one launch, whose workgroups each compute all of p. It has to
    stop where p or the workgroups get many: tall, narrow layers once took it with a workgroup for each column of x."""
    n = ctypes.c_int64()

    def one(M, K, N):
        assert lib.dgnn_linear_backward_workspace(M, K, N, 0, 2, ctypes.byref(n)) == 0
        return n.value == 0
    assert all(one(*s) for s in ((1, 602, 256), (8, 4096, 16), (64, 1433, 16), (1024, 256, 4), (1, 1, 1)))
    assert not any(one(*s) for s in ((4096, 1024, 1), (4096, 4096, 1), (1024, 4096, 1), (2048, 1500, 2), (64, 64, 64), (256, 100, 16), (8, 602, 512), (1, 4096, 4096)))
