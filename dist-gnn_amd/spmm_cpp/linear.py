"""The layer transform with its epilogue, y = act(x W + b) + r, and its gradients (C ABI: dgnn_linear_*, include/dgnn_train.h).

The reference's layers are ``torch.mm`` and a separate ReLU (light_dist_gnn/models/gcn.py:41,69-71); here bias, activation and
skip connection are part of the product, forward and backward. ``linear`` is the differentiable operator; the single
passes are there for layers with something in between (a GCN layer aggregates the output gradient before the products).

Matrices are 2-D, rows unit-stride (any distance between rows), of one type: fp32, bf16 or fp16. fp32 results are as close
to the exact sums as fp32 arithmetic is; with 16-bit types the gradient behind gelu or silu is rounded to the type before its
products, as a 16-bit tensor between two operations would be (not in ``linear``'s weight gradients of narrow layers, up to 64
columns, its input gradients of up to 2048 values and its backward pass of small layers). The order of the sums depends on the sizes alone, so runs agree to the bit.
There is no second derivative, no forward-mode derivative and no torch.jit.trace: each is an error. Calls can be captured in a
graph; as with every torch operator, ``backward()`` of a captured call needs leaves that no live eager graph holds, whose accumulation
belongs to the eager stream.
Checks, outputs, workspaces and the autograd node are in csrc/dgnn_torch.cpp; errors are RuntimeError.
"""
import torch

from . import _ext

ACTIVATIONS = {'none': 0, 'relu': 1, 'gelu': 2, 'silu': 3}           # DGNN_ACT_*


def _code(activation):
    try:
        return ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise RuntimeError(f'spmm_cpp.linear: unknown activation {activation!r} ({" | ".join(ACTIVATIONS)})') from None


def _call(f, *args):
    try:
        return f(*args)
    except TypeError:
        bad = [type(a).__name__ for a in args if not (a is None or isinstance(a, (torch.Tensor, int)))]
        raise RuntimeError(f'spmm_cpp.linear: an operand must be a torch.Tensor (got {", ".join(bad) or "None"})') from None


def linear(x, weight, bias=None, activation='none', residual=None):
    """y = act(x W + b) + r in one pass over x, differentiable (once) in x, weight, bias and residual.

    x [M, K], weight [K, N] (the layout of the models' weights), bias [N], residual [M, N]; activation 'none', 'relu', 'gelu'
    (with erf) or 'silu'. Rows unit-stride; x may be a view of padded rows (``row_padded``). M = 0 and K = 0 are allowed."""
    return _call(_ext.linear, x, weight, bias, _code(activation), residual)


def linear_forward(x, weight, bias=None, activation='none', residual=None, save=False):
    """(y, saved): y = act(x W + b) + r and, with ``save``, what ``linear_slope`` needs (None for 'none'): one bit per value
    for relu (int32 [M, ceil(N / 32)]), x W + b itself, in fp32, for gelu and silu."""
    return _call(_ext.linear_forward, x, weight, bias, _code(activation), residual, save)


def linear_slope(dy, saved, activation, need_bias=True):
    """(p, db): p = dy act'(x W + b), from what ``linear_forward`` saved, and the sums of p's columns (None unless
    ``need_bias``). For 'none' p is dy itself."""
    return _call(_ext.linear_slope, dy, saved, _code(activation), need_bias)


def linear_grad_input(p, weight, add=None):
    """dx = p W^T + add; ``add`` is what else reaches x, the gradient of a skip connection."""
    return _call(_ext.linear_grad_input, p, weight, add)


def linear_grad_weight(x, p):
    """dW = x^T p."""
    return _call(_ext.linear_grad_weight, x, p)
