"""AdamW's refusals and its C entry's checks (no GPU needed: nothing is launched)."""
import ctypes

import pytest
import torch

import numpy as np

import spmm_cpp

_TENSOR = np.dtype([('param', np.uint64), ('grad', np.uint64), ('numel', np.int64), ('start', np.int64), ('decay', np.float32),
                    ('rate', np.float32), ('root', np.float32), ('turn', np.uint32), ('index', np.int32), ('reserved', np.int32)])


class _CState(ctypes.Structure):          # struct dgnn_adamw_state (include/dgnn_train.h)
    _fields_ = [(n, ctypes.c_void_p) for n in ('exp_avg', 'exp_avg_sq', 'exp_avg_scale', 'exp_avg_sq_scale', 'master',
                                               'steps', 'factors')]


def _table(numel=4, start=0, param=1 << 20, grad=1 << 21, index=0):
    t = np.zeros(1, dtype=_TENSOR)
    t['numel'], t['start'], t['param'], t['grad'], t['index'] = numel, start, param, grad, index
    return t


def _call(table, state=None, dtype=0, bits=32, lr=0.1, b1=0.9, b2=0.9, eps=1e-8, count=None):
    if state is None:
        state = _CState(exp_avg=1 << 22, exp_avg_sq=1 << 23)
    return spmm_cpp.lib.dgnn_adamw(table.ctypes.data if table is not None else None, 1 if count is None else count, dtype, bits,
                                   ctypes.byref(state) if state else None, lr, b1, b2, eps, None)


@pytest.mark.parametrize('kw', [
    dict(table=None), dict(table=_table(), dtype=7), dict(table=_table(), bits=16), dict(table=_table(), lr=-1.0),
    dict(table=_table(), lr=float('nan')), dict(table=_table(), b1=1.0), dict(table=_table(), b2=-0.1), dict(table=_table(), eps=-1e-8),
    dict(table=_table(), state=_CState()), dict(table=_table(), state=_CState(exp_avg=1 << 22)),
    dict(table=_table(), bits=8),                                                     # no scales
    dict(table=_table(), state=_CState(exp_avg=(1 << 22) + 4, exp_avg_sq=1 << 23)),
    dict(table=_table(), state=_CState(exp_avg=1 << 22, exp_avg_sq=1 << 23, steps=1 << 24)),
    dict(table=_table(numel=-1)), dict(table=_table(start=128)), dict(table=_table(start=-256)), dict(table=_table(param=0)),
    dict(table=_table(grad=0)), dict(table=_table(param=(1 << 20) + 2)), dict(table=_table(grad=(1 << 20) + 1), dtype=1),
    dict(table=_table(), count=-1),
    dict(table=_table(index=-1), state=_CState(exp_avg=1 << 22, exp_avg_sq=1 << 23, steps=1 << 24, factors=1 << 25)),
])
def test_c_entry_refuses(kw):
    assert _call(**kw) == 1 and b'adamw' in spmm_cpp.lib.dgnn_last_error()


def test_c_entry_has_nothing_to_do():
    assert _call(_table(), count=0) == 0
    assert _call(_table(numel=0, param=0, grad=0), state=_CState()) == 0


@pytest.mark.parametrize('kw', [dict(lr=-1.0), dict(lr=float('nan')), dict(lr=float('inf')), dict(lr=torch.tensor(0.1)), dict(betas=(1.0, 0.9)),
                                dict(betas=(0.9,)), dict(betas=(0.9, -0.1)), dict(eps=-1.0), dict(weight_decay=-0.1), dict(state_bits=16)])
def test_arguments_refused(kw):
    with pytest.raises(ValueError, match='AdamW'):
        spmm_cpp.AdamW([torch.nn.Parameter(torch.ones(3))], **kw)


def test_cpu_parameters_refused():
    with pytest.raises(RuntimeError, match='no CPU path'):
        spmm_cpp.AdamW([torch.nn.Parameter(torch.ones(3))])


def test_header_and_signatures_agree():
    import os
    import re
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    txt = open(os.path.join(root, 'include', 'dgnn_train.h')).read()
    txt = re.sub(r'/\*.*?\*/', '', txt, flags=re.S)
    protos = {m.group(1): m.group(2) for m in re.finditer(r'\b(dgnn_[a-z0-9_]+)\s*\(([^)]*)\)\s*;', txt)}
    assert set(protos) == set(spmm_cpp._TRAIN_SIGNATURES)
    for name, args in spmm_cpp._TRAIN_SIGNATURES.items():
        assert protos[name].count(',') + 1 == len(args), name
        assert hasattr(spmm_cpp.lib, name)
