"""The expert-layer calls of the C++ Handle mirror
(cublas-rs_b200/examples/expert_example.cpp): exact products of whole numbers
in both types, and refusals."""
import os
import subprocess

import pytest

from conftest import PKG

pytestmark = pytest.mark.gpu


def test_cpp_expert_example():
    exe = os.path.join(PKG, "examples", "expert_example")
    if not os.path.exists(exe):
        subprocess.run(["make", "-C", PKG, "examples/expert_example"], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "all OK" in r.stdout
