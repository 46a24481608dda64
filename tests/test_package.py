"""The package and its build where torch is missing or is not the ROCm one."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

PKG = Path(__file__).resolve().parent.parent / "ssla-rt_amd"


def python(code, **env):
    return subprocess.run([sys.executable, "-c", code], env=dict(os.environ, PYTHONPATH=str(PKG), **env),
                          capture_output=True, text=True)


def test_everything_is_imported_without_torch():
    r = python("import sys; sys.modules['torch'] = None\nfrom ssla_hip import *\nprint(abi.SSLA_OK, lib.SSLA_OK, "
               "hybrid.__name__, 'ops' in globals())")
    assert r.returncode == 0, r.stderr
    assert r.stdout.split() == ["0", "0", "ssla_hip.hybrid", "False"]


def test_everything_includes_the_operators_where_they_are_built():
    pytest.importorskip("torch")
    r = python("from ssla_hip import *\nprint(ops.__name__)")
    assert r.returncode == 0 and r.stdout.split() == ["ssla_hip.ops"], r.stderr


def targets(path):
    """Whether `make` in the package would build the operators' module, with
    `path` in front of Python's."""
    r = subprocess.run(["make", "-n", "-B", "-C", str(PKG)], capture_output=True, text=True,
                       env=dict(os.environ, PYTHONPATH=str(path)))
    assert r.returncode == 0 and "libssla_hip.so" in r.stdout, r.stderr
    return "_ops.so" in r.stdout


def test_the_module_is_built_against_a_rocm_torch_only(tmp_path):
    assert targets(tmp_path)
    (tmp_path / "torch" / "lib").mkdir(parents=True)
    (tmp_path / "torch" / "__init__.py").write_text("")
    (tmp_path / "torch" / "lib" / "libtorch_cpu.so").write_text("")
    assert not targets(tmp_path)
