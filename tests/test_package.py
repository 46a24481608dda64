"""The package where torch is missing."""
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
