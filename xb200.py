"""Makes ``import xb200`` work from the repository's root.

The package lies in ``triton-xdna_b200/``, which is no importable name.  With
the root on ``sys.path`` this module is found under the package's name and
puts the package in its own place; with ``triton-xdna_b200/`` on the path
(before or after the root) the package is the same.
"""

import importlib.util
import os
import sys

_folder = os.path.join(os.path.dirname(os.path.abspath(__file__)), "triton-xdna_b200", "xb200")
_spec = importlib.util.spec_from_file_location(__name__, os.path.join(_folder, "__init__.py"),
                                               submodule_search_locations=[_folder])
sys.modules[__name__] = _package = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(_package)
