"""What make would build, with and without torch for its python3 (nothing is built here)."""
import os
import shutil
import subprocess
import sys

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vllm-ascend910_b200", "csrc")


def _plan(py):
    if shutil.which("make") is None:
        pytest.skip("no make")
    r = subprocess.run(["make", "-n", "-B", "-C", CSRC, f"PY={py}"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    return r.stdout, r.stderr


def test_the_library_needs_no_torch():
    """-S: a python3 without site-packages.  The library is built, the short way from Python is left out."""
    out, err = _plan(f"{sys.executable} -S")
    assert "libw4a8_b200.so" in out and "_native.so" not in out
    assert "Traceback" not in err


def test_with_torch_the_short_way_is_built():
    pytest.importorskip("torch")
    out, _ = _plan(sys.executable)
    assert "libw4a8_b200.so" in out and "_native.so" in out
