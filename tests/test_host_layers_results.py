"""Results of the layer operators that repeat elements, on the CPU under sanitizers."""
import os
import shutil
import subprocess

import pytest

from test_host_sanitizers import CSRC, ENV, ROOT, SAN


def run_host_check(tmp_path, name):
    """builds tests/<name>.cpp with the entry points and plain loops in place of the kernels, and runs it"""
    exe = str(tmp_path / name)
    sources = [os.path.join(ROOT, "tests", name + ".cpp"), os.path.join(ROOT, "tests", "host_rt_stub.cpp")]
    sources += [os.path.join(CSRC, f) for f in ("layers.cpp", "tensor.cpp", "state.cpp", "layout.cpp")]
    r = subprocess.run(SAN + sources + ["-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([exe], capture_output=True, text=True, env=ENV, timeout=300)
    assert r.returncode == 0, (r.stdout + r.stderr)[-3000:]
    return r.stdout


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not found")
def test_results_that_repeat_elements_are_refused(tmp_path):
    assert "results of layers ok" in run_host_check(tmp_path, "host_layers_results_check")
