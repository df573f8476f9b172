"""Host-only sources under AddressSanitizer and UndefinedBehaviorSanitizer: the layout
rules and the expression rewriter driven by tests/host_fuzz.cpp with random views and
random expression text, and the tensor / storage / state bookkeeping driven by
tests/host_tensor_walk.cpp against a host-memory stand-in for the runtime layer
(tests/host_rt_stub.cpp, linked into that test program only).  Needs g++ only; no device
and no library build."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "cltorch_amd", "csrc")


SAN = ["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=undefined", "-static-libasan",
       "-D__HIP_PLATFORM_AMD__", "-I", "/opt/rocm/include", "-I", os.path.join(ROOT, "include"), "-I", CSRC]
ENV = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=0", UBSAN_OPTIONS="print_stacktrace=1")


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not found")
def test_tensor_bookkeeping_under_sanitizers(tmp_path):
    exe = str(tmp_path / "host_tensor_walk")
    cmd = SAN + [os.path.join(ROOT, "tests", "host_tensor_walk.cpp"), os.path.join(ROOT, "tests", "host_rt_stub.cpp"),
                 os.path.join(CSRC, "tensor.cpp"), os.path.join(CSRC, "state.cpp"), "-o", exe]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([exe, "8000"], capture_output=True, text=True, env=ENV, timeout=300)
    assert r.returncode == 0, (r.stdout + r.stderr)[-3000:]
    assert "iterations ok" in r.stdout


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not found")
def test_layer_entry_points_under_sanitizers(tmp_path):
    """cltorch_amd/csrc/layers.cpp with plain loops in place of its kernels: views, stand-ins, in-place forms and
    refusals of layer norm, linear layer and grouped products."""
    exe = str(tmp_path / "host_layers_check")
    cmd = SAN + [os.path.join(ROOT, "tests", "host_layers_check.cpp"), os.path.join(ROOT, "tests", "host_rt_stub.cpp"),
                 os.path.join(CSRC, "layers.cpp"), os.path.join(CSRC, "tensor.cpp"), os.path.join(CSRC, "state.cpp"),
                 os.path.join(CSRC, "layout.cpp"), "-o", exe]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([exe, "400"], capture_output=True, text=True, env=ENV, timeout=300)
    assert r.returncode == 0, (r.stdout + r.stderr)[-3000:]
    assert "rounds of layers ok" in r.stdout


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not found")
def test_layout_and_rewrite_under_sanitizers(tmp_path):
    inc = os.path.join(CSRC, "apply_device_src.inc")
    if not os.path.exists(inc):                      # generated by the library build
        from cltorch_amd import build
        build.embed_skeleton()
    exe = str(tmp_path / "host_fuzz")
    cmd = ["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=undefined", "-static-libasan",
           "-D__HIP_PLATFORM_AMD__", "-I", "/opt/rocm/include", "-I", os.path.join(ROOT, "include"), "-I", CSRC,
           os.path.join(ROOT, "tests", "host_fuzz.cpp"), os.path.join(ROOT, "tests", "test_hooks.cpp"),
           os.path.join(CSRC, "layout.cpp"), os.path.join(CSRC, "expr.cpp"),
           "-o", exe]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=0", UBSAN_OPTIONS="print_stacktrace=1")
    r = subprocess.run([exe, "20000"], capture_output=True, text=True, env=env, timeout=300)
    assert r.returncode == 0, (r.stdout + r.stderr)[-3000:]
    assert "iterations ok" in r.stdout


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not found")
@pytest.mark.parametrize("sanitizer", ["thread", "address,undefined"])
def test_host_copier_threads_and_piece_loops_under_sanitizers(tmp_path, sanitizer):
    """cltorch_amd/csrc/host_copiers.h (the copier threads, the piece loops of the staged copies, the upload ring)
    against host memory with a DMA that completes late: every piece boundary, counts on both sides of the
    thresholds, a failing transfer, two callers at once, shutdown and restart, and a forked child that copies."""
    exe = str(tmp_path / "host_copiers_check")
    cmd = ["g++", "-std=c++17", "-O1", "-g", f"-fsanitize={sanitizer}", "-fno-sanitize-recover=undefined", "-pthread", "-I", CSRC,
           os.path.join(ROOT, "tests", "host_copiers_check.cpp"), "-o", exe]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=0", UBSAN_OPTIONS="print_stacktrace=1", TSAN_OPTIONS="halt_on_error=1:die_after_fork=0")   # the forked child starts threads of its own
    r = subprocess.run([exe], capture_output=True, text=True, env=env, timeout=600)
    assert r.returncode == 0, (r.stdout + r.stderr)[-3000:]
    assert "host copiers ok" in r.stdout
