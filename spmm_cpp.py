"""``import spmm_cpp`` from the repository's root. The package lies in ``dist-gnn_amd/``, a name that no import statement can
spell: this module puts that folder on the path and gives its place to the package, so both ways in name the same module."""
import importlib
import os
import sys

_package = os.path.join(os.path.dirname(os.path.abspath(__file__)), 'dist-gnn_amd')
if sys.path[:1] != [_package]:
    sys.path.insert(0, _package)
del sys.modules[__name__]
importlib.import_module(__name__)
