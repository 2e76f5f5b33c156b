"""The drop-in path without libhomura_nn.so beside it: it imports and works, and what needs the library says which file is missing."""
import glob
import os
import shutil
import subprocess
import sys

import pytest

from homura_amd import capi

PACKAGE = os.path.dirname(os.path.abspath(capi.__file__))


@pytest.fixture()
def without(tmp_path):
    """The package with the libraries of the drop-in path only."""
    to = tmp_path / "homura_amd"
    (to / "lib").mkdir(parents=True)
    for name in ("__init__.py", "capi.py"):
        shutil.copy(os.path.join(PACKAGE, name), to / name)
    for path in glob.glob(os.path.join(PACKAGE, "_host*.so")):
        shutil.copy(path, to / os.path.basename(path))
    os.symlink(os.path.join(PACKAGE, "lib", "libhomura_rocm.so"), to / "lib" / "libhomura_rocm.so")
    return tmp_path


def run(at, program):
    return subprocess.run([sys.executable, "-c", program], cwd=at, capture_output=True, text=True, timeout=120,
                          env={k: v for k, v in os.environ.items() if k != "PYTHONPATH"})


def test_the_c_abi_without_it(without):
    r = run(without, "from homura_amd import capi\nprint(capi.lib.hmr_built_archs().decode())\n"
                     "try:\n    capi.nn\nexcept ImportError as e:\n    print('libhomura_nn.so' in str(e))\n"
                     "try:\n    capi.other\nexcept AttributeError:\n    print('no other')\n")
    assert r.returncode == 0 and r.stdout.split("\n")[:3] == ["gfx950", "True", "no other"], r.stderr


def test_the_host_layer_without_it(without):
    r = run(without, "import homura_amd\nh = homura_amd.load_host()\nprint(h.promote_types(h.DType.BF16, h.DType.F32))\n")
    assert r.returncode == 0 and "F32" in r.stdout, r.stderr


def test_the_module_has_it():
    assert capi.nn is capi.nn and capi.nn.hmn_last_error() is not None
