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
sys.exit(pytest.main(["-q", "-x", "--tb=short", "-p", "no:cacheprovider", "--noconftest", "-p", "lm_emulated_plugin"] + sys.argv[2:]))
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


def start(args, sms="2"):
    so = build_driver()
    env = dict(os.environ, GPUARRAY_NVRTC_PATH=so, GPUARRAY_CACHE_PATH="", SIMT_DIR=SIMT, SIMT_BUILD=BUILD,
               SIMT_TEMPLATES=os.path.join(ROOT, "libgpuarray_b200", "csrc", "templates"), SIMT_SMS=sms,
               PYTHONPATH=os.pathsep.join([ROOT, os.path.join(ROOT, "tests"), SIMT]))
    return subprocess.Popen([sys.executable, "-c", CHILD, so] + args, cwd=ROOT, env=env, stdout=subprocess.PIPE,
                            stderr=subprocess.STDOUT, text=True)


CASES = os.path.join(ROOT, "tests", "lm_operators_cases.py")
PARTS = {
    "embed": [CASES, "-k", "embed and not gradient"],
    "embed gradient": [CASES, "-k", "test_embed_gradient and not sorted and not strides and not broadcast"],
    "embed gradient, sorted": [CASES, "-k", "embed_gradient and (sorted or strides or broadcast)"],
    "log probabilities": [CASES, "-k", "logprobs and not gradient"],
    "log probabilities, gradient": [CASES, "-k", "logprobs and gradient"],
    "clip and all together": [CASES, "-k", "clip or together or another_context"],
    "captured": [os.path.join(SIMT, "capture_cases.py")],
}


@pytest.fixture(scope="module")
def children(built):
    """every part in a process of its own, side by side"""
    procs = {name: start(args) for name, args in PARTS.items()}
    yield procs
    for p in procs.values():
        if p.poll() is None:
            p.kill()
        p.communicate()


@pytest.mark.parametrize("part", list(PARTS))
def test_cases_under_the_emulator(children, part):
    out, _ = children[part].communicate(timeout=900)
    assert children[part].returncode == 0 and " passed" in out, out[-6000:]
