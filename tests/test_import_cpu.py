"""The package is found from the root of the repository as well as through PYTHONPATH, and it is the
same one."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "smoothquant-mixedprecision_amd")
PROGRAM = """
import sys
from smoothquant import experts, ops            # submodules first, by the package's name
import smoothquant, smoothquant.fake_quant as fq
from smoothquant import quantize_model
assert smoothquant.experts is experts and sys.modules["smoothquant.ops"] is ops
assert smoothquant.__name__ == "smoothquant" and smoothquant.__spec__.name == "smoothquant"
assert quantize_model is fq.quantize_model and fq.W4A4Linear.__module__ == "smoothquant.fake_quant"
print(smoothquant.__file__)
"""


@pytest.mark.parametrize("path,cwd", [(None, ROOT), (ROOT, os.path.dirname(ROOT)), (PKG, ROOT)])
def test_import_from_the_root(path, cwd):
    env = {k: v for k, v in os.environ.items() if k != "PYTHONPATH"}
    if path:
        env["PYTHONPATH"] = path
    r = subprocess.run([sys.executable, "-c", PROGRAM], cwd=cwd, env=env, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-1500:]
    assert os.path.realpath(r.stdout.split()[-1]) == os.path.realpath(
        os.path.join(PKG, "smoothquant", "__init__.py"))


def test_objects_travel_between_both_ways(tmp_path):
    """A module pickled by a program started at the root loads in one with the folder on the path."""
    f = str(tmp_path / "m.pt")
    env = {k: v for k, v in os.environ.items() if k != "PYTHONPATH"}
    save = f"import torch; from smoothquant.experts import W4A4Experts; torch.save(W4A4Experts('gelu'), {f!r})"
    load = f"import torch; m = torch.load({f!r}, weights_only=False); assert m.act == 'gelu'"
    for prog, e in ((save, env), (load, dict(env, PYTHONPATH=PKG))):
        r = subprocess.run([sys.executable, "-c", prog], cwd=ROOT if e is env else str(tmp_path), env=e,
                           capture_output=True, text=True)
        assert r.returncode == 0, r.stderr[-1500:]
