"""The layer transform with its epilogue, y = act(x W + b) + r, and its gradients (C ABI: dgnn_linear_*, include/dgnn_train.h).

The reference's layers are ``torch.mm`` and a separate ReLU (light_dist_gnn/models/gcn.py:41,69-71); here bias, activation and
skip connection are part of the product, forward and backward. ``linear`` is the differentiable operator; the single
passes are there for layers with something in between (a GCN layer aggregates the output gradient before the products).

Matrices are 2-D, rows unit-stride (any distance between rows), of one type: fp32, bf16 or fp16. fp32 results are as close
to the exact sums as fp32 arithmetic is; the order of the sums depends on the sizes alone, so runs agree to the bit.
"""
import ctypes

import torch

from . import _DTYPES, _check, _lib, _stream

ACTIVATIONS = {'none': 0, 'relu': 1, 'gelu': 2, 'silu': 3}           # DGNN_ACT_*
_FORWARD, _SLOPE, _GRAD_INPUT, _GRAD_WEIGHT = range(4)               # DGNN_LINEAR_*


def _rows(t, name, like=None, shape=None):
    """(pointer, elements between rows) of a 2-D operand; ``like``: the operand whose type and device it has to have."""
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f'spmm_cpp.linear: {name} must be a torch.Tensor')
    if not t.is_cuda:
        raise RuntimeError(f'spmm_cpp.linear: {name} is on {t.device}; this operator has no CPU path')
    if t.dtype not in _DTYPES:
        raise RuntimeError(f'spmm_cpp.linear: {name} must be fp32, bf16 or fp16, got {t.dtype}')
    if t.dim() != 2:
        raise RuntimeError(f'spmm_cpp.linear: {name} must have 2 dims, got {t.dim()}')
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        raise RuntimeError(f'spmm_cpp.linear: {name} is {t.dtype} on {t.device}, the other operands are {like.dtype} on {like.device}')
    if shape is not None and t.shape != shape:
        raise RuntimeError(f'spmm_cpp.linear: {name} is {tuple(t.shape)}, expected {tuple(shape)}')
    n, f = t.shape
    s0, s1 = t.stride()
    if f > 1 and s1 != 1:
        raise RuntimeError(f'spmm_cpp.linear: {name} must be row-major (stride(1) == 1)')
    if n <= 1:
        s0 = max(f, 1)
    elif s0 < f:
        raise RuntimeError(f'spmm_cpp.linear: {name} has overlapping rows')
    return t.data_ptr(), s0


def _vector(t, name, n, like):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dim() != 1 or t.numel() != n or t.dtype != like.dtype or t.device != like.device:
        raise RuntimeError(f'spmm_cpp.linear: {name} must be a vector of {n} {like.dtype} on {like.device}')
    if not t.is_contiguous():
        raise RuntimeError(f'spmm_cpp.linear: {name} must be contiguous')
    return t.data_ptr()


def _code(activation):
    try:
        return ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise RuntimeError(f'spmm_cpp.linear: unknown activation {activation!r} ({" | ".join(ACTIVATIONS)})') from None


def _workspace(kind, M, K, N, t):
    """The pass's workspace, from the caching allocator at every call: calls on different streams and captured graphs each
    have their own."""
    need = ctypes.c_int64()
    _check(_lib.dgnn_linear_workspace(kind, M, K, N, _DTYPES[t.dtype], ctypes.byref(need)), 'linear_workspace')
    if need.value == 0:
        return None, None, 0
    ws = torch.empty(need.value // 4, dtype=torch.float32, device=t.device)
    return ws, ws.data_ptr(), need.value


def linear_forward(x, weight, bias=None, activation='none', residual=None, save=False):
    """(y, saved): y = act(x W + b) + r and, with ``save``, what ``linear_slope`` needs (None for 'none'): one bit per value
    for relu (int32 [M, ceil(N / 32)]), x W + b itself for gelu and silu."""
    xp, ldx = _rows(x, 'x')
    wp, ldw = _rows(weight, 'weight', x)
    (M, K), N = x.shape, weight.shape[1]
    if weight.shape[0] != K:
        raise RuntimeError(f'spmm_cpp.linear: shape mismatch x{tuple(x.shape)} weight{tuple(weight.shape)}')
    act = _code(activation)
    bp = _vector(bias, 'bias', N, x)
    rp, ldr = (None, 0) if residual is None else _rows(residual, 'residual', x, (M, N))
    with torch.cuda.device(x.device):
        y = torch.empty(M, N, dtype=x.dtype, device=x.device)
        saved, sp, lds = None, None, 0
        if save and act:
            saved = torch.empty(M, -(-N // 32), dtype=torch.int32, device=x.device) if act == 1 else torch.empty_like(y)
            sp, lds = saved.data_ptr(), max(saved.shape[1], 1)
        if M and N:
            ws, wsp, nbytes = _workspace(_FORWARD, M, K, N, x)
            _check(_lib.dgnn_linear_forward(xp, ldx, wp, ldw, bp, rp, ldr, y.data_ptr(), N, sp, lds, M, K, N, _DTYPES[x.dtype], act,
                                            wsp, nbytes, _stream(x)), 'linear_forward')
    return y, saved


def linear_slope(dy, saved, activation, need_bias=True):
    """(p, db): p = dy act'(x W + b), from what ``linear_forward`` saved, and the sums of p's columns (None unless
    ``need_bias``). For 'none' p is dy itself."""
    dp, ldd = _rows(dy, 'dy')
    act = _code(activation)
    M, N = dy.shape
    sp, lds = None, 0
    if act:
        if not isinstance(saved, torch.Tensor) or not saved.is_contiguous() or saved.device != dy.device:
            raise RuntimeError('spmm_cpp.linear: saved must be what linear_forward returned')
        want = ((M, -(-N // 32)), torch.int32) if act == 1 else ((M, N), dy.dtype)
        if tuple(saved.shape) != want[0] or saved.dtype != want[1]:
            raise RuntimeError(f'spmm_cpp.linear: saved must be {want[1]} {want[0]} for {activation}, got {saved.dtype} {tuple(saved.shape)}')
        sp, lds = saved.data_ptr(), max(saved.shape[1], 1)
    if not act and not need_bias:
        return dy, None
    with torch.cuda.device(dy.device):
        p = torch.empty(M, N, dtype=dy.dtype, device=dy.device) if act else None
        db = torch.empty(N, dtype=dy.dtype, device=dy.device) if need_bias else None
        ws, wsp, nbytes = _workspace(_SLOPE, M, 0, N, dy) if need_bias else (None, None, 0)
        _check(_lib.dgnn_linear_slope(dp, ldd, sp, lds, None if p is None else p.data_ptr(), N, None if db is None else db.data_ptr(),
                                      M, N, _DTYPES[dy.dtype], act, wsp, nbytes, _stream(dy)), 'linear_slope')
    return (dy if p is None else p), db


def linear_grad_input(p, weight, add=None):
    """dx = p W^T + add; ``add`` is what else reaches x, the gradient of a skip connection."""
    pp, ldp = _rows(p, 'p')
    wp, ldw = _rows(weight, 'weight', p)
    (M, N), K = p.shape, weight.shape[0]
    if weight.shape[1] != N:
        raise RuntimeError(f'spmm_cpp.linear: shape mismatch p{tuple(p.shape)} weight{tuple(weight.shape)}')
    ap, lda = (None, 0) if add is None else _rows(add, 'add', p, (M, K))
    with torch.cuda.device(p.device):
        dx = torch.empty(M, K, dtype=p.dtype, device=p.device)
        if M and K:
            ws, wsp, nbytes = _workspace(_GRAD_INPUT, M, K, N, p)
            _check(_lib.dgnn_linear_grad_input(pp, ldp, wp, ldw, ap, lda, dx.data_ptr(), K, M, K, N, _DTYPES[p.dtype], wsp, nbytes,
                                               _stream(p)), 'linear_grad_input')
    return dx


def linear_grad_weight(x, p):
    """dW = x^T p."""
    xp, ldx = _rows(x, 'x')
    pp, ldp = _rows(p, 'p', x)
    (M, K), N = x.shape, p.shape[1]
    if p.shape[0] != M:
        raise RuntimeError(f'spmm_cpp.linear: shape mismatch x{tuple(x.shape)} p{tuple(p.shape)}')
    with torch.cuda.device(x.device):
        dw = torch.empty(K, N, dtype=x.dtype, device=x.device)
        if K and N:
            ws, wsp, nbytes = _workspace(_GRAD_WEIGHT, M, K, N, x)
            _check(_lib.dgnn_linear_grad_weight(xp, ldx, pp, ldp, dw.data_ptr(), N, M, K, N, _DTYPES[x.dtype], wsp, nbytes, _stream(x)),
                   'linear_grad_weight')
    return dw


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        wanted = ctx.needs_input_grad
        y, saved = linear_forward(x, weight, bias, activation, residual, save=any(wanted[:3]))
        ctx.save_for_backward(x if wanted[1] else None, weight if wanted[0] else None, saved)
        ctx.act, ctx.K = ACTIVATIONS[activation], x.shape[1]
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, saved = ctx.saved_tensors
        want_x, want_w, want_b, want_r = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if want_x or want_w or want_b:
            # one call for all of them (x, weight and saved were checked when they were saved; dy is of y's shape and type)
            (M, N), K, act = dy.shape, ctx.K, ctx.act
            ldd, s1 = dy.stride()
            if s1 != 1 and N > 1 or ldd < N and M > 1:                # an expanded or transposed gradient
                dy = dy.contiguous()
                ldd = N
            dtype, dev = dy.dtype, dy.device
            code = _DTYPES[dtype]
            with torch.cuda.device(dev):
                need = ctypes.c_int64()
                _check(_lib.dgnn_linear_backward_workspace(M, K, N, code, act, ctypes.byref(need)), 'linear_backward')
                ws = torch.empty(need.value, dtype=torch.uint8, device=dev)
                xp = wp = dxp = dwp = dbp = sp = None
                ldx = ldw = lds = 0
                if want_x:
                    dx = torch.empty((M, K), dtype=dtype, device=dev)
                    dxp, wp, ldw = dx.data_ptr(), weight.data_ptr(), weight.stride(0) if K > 1 else max(N, 1)
                if want_w:
                    dw = torch.empty((K, N), dtype=dtype, device=dev)
                    dwp, xp, ldx = dw.data_ptr(), x.data_ptr(), x.stride(0) if M > 1 else max(K, 1)
                if want_b:
                    db = torch.empty(N, dtype=dtype, device=dev)
                    dbp = db.data_ptr()
                if saved is not None:
                    sp, lds = saved.data_ptr(), max(saved.shape[1], 1)
                _check(_lib.dgnn_linear_backward(xp, ldx, wp, ldw, dy.data_ptr(), max(ldd, N) if M > 1 else max(N, 1), sp, lds, dxp, max(K, 1), dwp,
                                                 max(N, 1), dbp, M, K, N, code, act, ws.data_ptr(), need.value, _stream(dy)), 'linear_backward')
        return dx, dw, db, dy if want_r else None, None


def linear(x, weight, bias=None, activation='none', residual=None):
    """y = act(x W + b) + r in one pass over x, differentiable in x, weight, bias and residual.

    x [M, K], weight [K, N] (the layout of the models' weights), bias [N], residual [M, N]; activation 'none', 'relu', 'gelu'
    (with erf) or 'silu'. Rows unit-stride; x may be a view of padded rows (``row_padded``). M = 0 and K = 0 are allowed."""
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (x, weight, bias, residual)):
        return _Linear.apply(x, weight, bias, residual, activation)
    return linear_forward(x, weight, bias, activation, residual)[0]
