"""`import smoothquant` from the root of the repository.

The package lies in smoothquant-mixedprecision_amd/ (no name that Python imports); with the root
first on the path, as for a program started there, this file stands for it: the name is bound to
the package itself, the same modules as with that folder on PYTHONPATH.
"""
import importlib.util
import os
import sys

_folder = os.path.join(os.path.dirname(os.path.abspath(__file__)),
                       "smoothquant-mixedprecision_amd", "smoothquant")
_spec = importlib.util.spec_from_file_location(
    __name__, os.path.join(_folder, "__init__.py"), submodule_search_locations=[_folder])
_package = importlib.util.module_from_spec(_spec)
sys.modules[__name__] = _package
_spec.loader.exec_module(_package)
