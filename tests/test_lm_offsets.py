"""The byte offset of a token or row from its number, as the language-model
kernels compute it (ga__lm_offset of ga_lm_common.cuh), compiled for the host
and compared with divisions of whole numbers around the places where it changes
from 32-bit to 64-bit arithmetic."""
import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SIMT = os.path.join(ROOT, "tests", "simt")
TEMPLATES = os.path.join(ROOT, "libgpuarray_b200", "csrc", "templates")

SOURCE = """
#include "ga_lm_common.cuh"
extern "C" long long offset(int nd, unsigned long long i, const unsigned long long *dims, const long long *strs) {
  if (i < 0x80000000ULL) { /* an index of 32 bits */
    const unsigned int j = (unsigned int)i;
    const long long p = nd == 1 ? ga__lm_offset<1>(j, dims, strs) : nd == 2 ? ga__lm_offset<2>(j, dims, strs)
                      : nd == 3 ? ga__lm_offset<3>(j, dims, strs) : ga__lm_offset<4>(j, dims, strs);
    const long long q = nd == 1 ? ga__lm_offset<1>(i, dims, strs) : nd == 2 ? ga__lm_offset<2>(i, dims, strs)
                      : nd == 3 ? ga__lm_offset<3>(i, dims, strs) : ga__lm_offset<4>(i, dims, strs);
    return p == q ? p : -1;
  }
  return nd == 1 ? ga__lm_offset<1>(i, dims, strs) : nd == 2 ? ga__lm_offset<2>(i, dims, strs)
       : nd == 3 ? ga__lm_offset<3>(i, dims, strs) : ga__lm_offset<4>(i, dims, strs);
}
"""


@pytest.fixture(scope="module")
def offset(tmp_path_factory):
    d = tmp_path_factory.mktemp("offset")
    src, so = str(d / "offset.cpp"), str(d / "offset.so")
    with open(src, "w") as f:
        f.write(SOURCE)
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-w", "-include", "ga_lm_ptx.cuh", "-I", os.path.join(SIMT, "include"),
                        "-I", TEMPLATES, src, os.path.join(SIMT, "simt_runtime.cpp"), os.path.join(SIMT, "simt_cluster.cpp"), "-o", so],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    f = ctypes.CDLL(so).offset
    f.restype = ctypes.c_longlong

    def call(i, dims, strs):
        return f(len(dims), ctypes.c_ulonglong(i), (ctypes.c_ulonglong * 4)(*dims), (ctypes.c_longlong * 4)(*strs))
    return call


W = 1 << 32


@pytest.mark.parametrize("dims", [(5,), (3 * W,), (2, 7), (2, W - 2), (2, W - 1), (2, W), (2, W + 1), (W, 2), (W + 3, 3), (2, 3, W + 5), (2, W + 5, 1),
                                  (3, 2, 5, W - 1), (2, 2, 2, 2 * W)], ids=str)
def test_offsets_around_32_bits(offset, dims):
    strs = [-7, 1 << 33, 12, 2][4 - len(dims):]
    count = 1
    for n in dims:
        count *= n
    for i in {0, 1, 2, 6, W // 2, W - 3, W - 2, W - 1, W, W + 1, 2 * W - 1, 2 * W, count // 2, count - 1}:
        if i >= count:
            continue
        want, r = 0, i
        for n, s in list(zip(dims, strs))[:0:-1]:
            want += r % n * s
            r //= n
        want += r * strs[0]
        assert offset(i, dims, strs) == want, (i, dims)
