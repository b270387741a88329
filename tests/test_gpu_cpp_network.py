"""The attribute network's operators through the C++ interface (tests/cpp/network_step.cpp)."""
import os
import subprocess

import pytest

from tinygs_amd import build as hb

pytestmark = pytest.mark.gpu


def test_cpp_network_step(hip):
    exe = hb.cpp_test_bin("network_step")
    if not os.path.exists(exe):
        hb.build_cpp_test(verbose=False)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "network ok" in r.stdout
