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
