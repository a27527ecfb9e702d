"""`make` in csrc/, without the package's build function."""
import os
import subprocess

import pytest

from conftest import ROOT


def test_make_finds_what_the_extension_needs():
    pytest.importorskip("torch")
    env = {k: v for k, v in os.environ.items() if not k.startswith("EXT_")}
    r = subprocess.run(["make", "-n", "-B", "-C", os.path.join(ROOT, "spmspm_b200", "csrc"), "../_torch_ext.so"], capture_output=True, text=True, env=env)
    assert r.returncode == 0, r.stderr
    command = next(line for line in r.stdout.splitlines() if "torch_ext.cpp" in line)
    assert "torch/include" in command and "_GLIBCXX_USE_CXX11_ABI=" in r.stdout and "torch/lib" in r.stdout
