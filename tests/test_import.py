"""Ways to `spmm_cpp` from a fresh interpreter."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _run(code, cwd=ROOT, path=''):
    env = {k: v for k, v in os.environ.items() if k != 'PYTHONPATH'}
    if path:
        env['PYTHONPATH'] = path
    r = subprocess.run([sys.executable, '-c', code], cwd=cwd, env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    return r.stdout


@pytest.mark.parametrize('first', ['import spmm_cpp', 'from spmm_cpp import AdamW, linear, spmm_cusparse', 'import spmm_cpp.adamw'])
def test_import_from_the_repository_root(first, tmp_path):
    """The root on the path is enough, whether by the working folder or by PYTHONPATH, and it is the one package."""
    code = first + '\nimport sys, spmm_cpp, os\nprint(os.path.realpath(spmm_cpp.__file__))\nassert spmm_cpp.linear and spmm_cpp.spmm_cusparse\n' \
        'import models.gcn\nassert sys.modules["spmm_cpp"] is spmm_cpp and spmm_cpp.adamw.AdamW is spmm_cpp.AdamW'
    want = os.path.join(ROOT, 'dist-gnn_amd', 'spmm_cpp', '__init__.py')
    assert _run(code).strip() == want
    assert _run(code, cwd=tmp_path, path=ROOT).strip() == want
    assert _run(code, cwd=os.path.join(ROOT, 'dist-gnn_amd'), path=ROOT).strip() == want


def test_the_spmm_does_not_need_the_torch_binding():
    """The binding of the training operators is loaded at their first use; without it they alone fail, and say how to build it."""
    code = '''
import sys, spmm_cpp, models.gcn, torch
def loaded():
    return any('_dgnn_torch' in line for line in open('/proc/self/maps'))
assert not loaded()
x = torch.ones(2, 2)
try:
    spmm_cpp.spmm_cusparse(x, x, x, 2, 2, x, x, 1, 1)
except RuntimeError:
    pass
kept, spmm_cpp._TORCH_LIB_PATH = spmm_cpp._TORCH_LIB_PATH, sys.argv[1]
for call in (lambda: spmm_cpp.linear(x, x), lambda: spmm_cpp.linear_grad_weight(x, x)):
    try:
        call()
        raise SystemExit('no error')
    except RuntimeError as e:
        assert '_dgnn_torch' in str(e) and '__graft_entry__' in str(e), e
assert not loaded()
spmm_cpp._TORCH_LIB_PATH = kept
try:
    spmm_cpp.linear(x, x)
except RuntimeError as e:
    assert 'no CPU path' in str(e), e
assert loaded()
'''
    for path in ('/nowhere/_dgnn_torch.so', os.path.join(ROOT, 'dist-gnn_amd', 'lib', 'libdgnn_spmm.so')):
        r = subprocess.run([sys.executable, '-c', code.replace('sys.argv[1]', repr(path)).replace("'_dgnn_torch' in str(e) and ", '')],
                           cwd=os.path.join(ROOT, 'dist-gnn_amd'), capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stderr[-2000:]
