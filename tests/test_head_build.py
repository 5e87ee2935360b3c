"""CPU tests of the build: what `make` would run, with and without a torch to bind to."""
import os
import subprocess
import sys

from conftest import PKG_NAME, ROOT


def _commands(*args):
    return subprocess.run(["make", "-n", "-B", "-C", os.path.join(ROOT, PKG_NAME, "csrc"), *args], check=True, capture_output=True,
                          text=True).stdout


def test_the_library_needs_no_torch():
    both = _commands("PYTHON=" + sys.executable)
    assert "head_binding.cpp" in both and "vocab_loss.hip" in both
    for args in (["PYTHON=false"], ["lib", "PYTHON=" + sys.executable], ["lib", "PYTHON=false"]):
        out = _commands(*args)
        assert "head_binding.cpp" not in out and "-shared -fPIC -o ../libadvpatch_hip.so" in out
