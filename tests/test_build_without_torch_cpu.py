"""The library and the pybind module need no torch: where Python cannot import it, both builds leave the
torch front end out and make the rest, as they did before it was there.  CPU only; nothing is compiled."""
import os
import shutil
import subprocess
import sys

import pytest

from tests.conftest import ROOT


@pytest.fixture
def no_torch(tmp_path):
    """An environment in which `import torch` fails."""
    (tmp_path / "path" / "torch").mkdir(parents=True)
    (tmp_path / "path" / "torch" / "__init__.py").write_text("raise ImportError('no torch here')\n")
    return dict(os.environ, PYTHONPATH=str(tmp_path / "path"))


def test_the_environment_has_no_torch(no_torch):
    assert subprocess.run([sys.executable, "-c", "import torch"], env=no_torch, capture_output=True).returncode != 0


@pytest.mark.skipif(shutil.which("cmake") is None or shutil.which("ninja") is None, reason="cmake and ninja are needed")
def test_cmake_configures_the_library_without_torch(no_torch, tmp_path):
    def targets(env, name):
        b = str(tmp_path / name)
        r = subprocess.run(["cmake", "-S", ROOT, "-B", b, "-G", "Ninja"], capture_output=True, text=True, env=env, timeout=300)
        assert r.returncode == 0, r.stdout + r.stderr
        r = subprocess.run(["ninja", "-C", b, "-t", "targets", "all"], capture_output=True, text=True, timeout=60)
        return r.stdout
    without, with_torch = targets(no_torch, "without"), targets(os.environ, "with")
    assert "libnmi.so" in without and "nmi_binding" in without and "nmi_front" not in without
    assert "libnmi.so" in with_torch and "nmi_binding" in with_torch and "nmi_front" in with_torch


def test_build_py_leaves_the_front_end_out_without_torch(no_torch):
    code = "from nemotron_infer_amd import build\nassert build.build_front() is None\nassert build.build_front(verbose=True) is None"
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, env=no_torch, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    assert "left out" in r.stdout
