"""CPU: the C library's build does not need torch."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "stable-diffusion_amd", "csrc")


@pytest.mark.skipif(shutil.which("make") is None, reason="no make")
def test_default_goal_leaves_the_torch_module_out_where_there_is_no_torch(tmp_path):
    fake = tmp_path / "python"
    fake.write_text("#!/bin/sh\necho 'No module named torch' >&2\nexit 1\n")
    fake.chmod(0o755)

    def plan(*goal):
        return subprocess.run(["make", "-n", "-B", "-C", CSRC, f"PYTHON={fake}", *goal], stdout=subprocess.PIPE,
                              stderr=subprocess.STDOUT, text=True)
    r = plan()
    assert r.returncode == 0 and "libsdmi.so" in r.stdout and "torch_layers.cpp" not in r.stdout, r.stdout[-2000:]
    assert plan("layers").returncode != 0                 # asked for by name it is an error


@pytest.mark.skipif(shutil.which("make") is None, reason="no make")
def test_default_goal_builds_both_where_torch_is():
    r = subprocess.run(["make", "-n", "-B", "-C", CSRC, "PYTHON=python3"], stdout=subprocess.PIPE, stderr=subprocess.STDOUT,
                       text=True)
    assert r.returncode == 0 and "libsdmi.so" in r.stdout and "torch_layers.cpp" in r.stdout
