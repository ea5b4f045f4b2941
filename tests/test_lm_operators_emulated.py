"""The language-model operators on the CPU: the library's host code and its
kernel templates run as they are, over a stand-in for the CUDA driver
(tests/simt/fake_cuda.cpp) that executes kernels with the SIMT emulator and
puts every allocation before an inaccessible page. The cases run in a child
process, because a process binds the driver once."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SIMT = os.path.join(ROOT, "tests", "simt")
BUILD = os.path.join(ROOT, "libgpuarray_b200", "build", "simt")

CHILD = """
import ctypes, os, sys
ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)   # the stand-in answers to libcuda.so.1
import pytest
sys.exit(pytest.main(["-q", "-x", "-p", "no:cacheprovider", "--noconftest", "-p", "lm_emulated_plugin"] + sys.argv[2:]))
"""


def build_driver():
    so = os.path.join(BUILD, "libcuda.so.1")
    src = os.path.join(SIMT, "fake_cuda.cpp")
    os.makedirs(BUILD, exist_ok=True)
    if not os.path.exists(so) or os.path.getmtime(so) < os.path.getmtime(src):
        tmp = "%s.%d" % (so, os.getpid())
        r = subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-w", "-I/usr/local/cuda/include",
                            "-Wl,-soname,libcuda.so.1", src, "-o", tmp, "-ldl"], capture_output=True, text=True)
        assert r.returncode == 0, r.stderr[-3000:]
        os.replace(tmp, so)
    return so


def run(args, sms="2"):
    so = build_driver()
    env = dict(os.environ, GPUARRAY_NVRTC_PATH=so, GPUARRAY_CACHE_PATH="", SIMT_DIR=SIMT, SIMT_BUILD=BUILD,
               SIMT_TEMPLATES=os.path.join(ROOT, "libgpuarray_b200", "csrc", "templates"), SIMT_SMS=sms,
               PYTHONPATH=os.pathsep.join([ROOT, os.path.join(ROOT, "tests"), SIMT]))
    r = subprocess.run([sys.executable, "-c", CHILD, so] + args, cwd=ROOT, env=env, capture_output=True,
                       text=True, timeout=900)
    assert r.returncode == 0, (r.stdout + r.stderr)[-6000:]
    return r.stdout


@pytest.mark.parametrize("part", ["embed", "logprobs", "clip or together or another_context"])
def test_cases_under_the_emulator(built, part):
    out = run([os.path.join(ROOT, "tests", "lm_operators_cases.py"), "-k", part])
    assert " passed" in out


def test_refusals_while_a_graph_is_captured(built):
    out = run([os.path.join(SIMT, "capture_cases.py")])
    assert " passed" in out
