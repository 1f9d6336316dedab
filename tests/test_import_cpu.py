"""The package is imported from the repository's root, as a program beside it does."""

import os
import subprocess
import sys

import pytest

from conftest import PKG_ROOT, ROOT

HERE = os.path.join(PKG_ROOT, "xb200", "__init__.py")


@pytest.mark.parametrize("paths", [[ROOT], [ROOT, PKG_ROOT], [PKG_ROOT, ROOT], [PKG_ROOT]])
def test_import_from(paths, tmp_path):
    code = (f"import sys; sys.path[:0] = {paths!r}\n"
            "from xb200 import ops\n"
            "import xb200, xb200.paged, xb200._lib\n"
            "from xb200 import XbError\n"
            "assert xb200.ops is ops and sys.modules['xb200'] is xb200 and XbError is xb200._lib.XbError\n"
            "xb200._lib.load()\n"
            "print(xb200.__file__)")
    env = {k: v for k, v in os.environ.items() if k != "PYTHONPATH"}
    got = subprocess.run([sys.executable, "-c", code], cwd=tmp_path, env=env, capture_output=True, text=True)
    assert got.returncode == 0, got.stderr
    assert os.path.realpath(got.stdout.strip()) == os.path.realpath(HERE)


def test_import_with_the_root_as_the_working_folder():
    """Nothing on the path but what Python puts there itself."""
    env = {k: v for k, v in os.environ.items() if k != "PYTHONPATH"}
    got = subprocess.run([sys.executable, "-c", "from xb200 import ops, paged"], cwd=ROOT, env=env, capture_output=True,
                         text=True)
    assert got.returncode == 0, got.stderr
