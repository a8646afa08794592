"""The attention's and the append's index rules at the ends of their ranges (the HIP-free headers of torq-tile_amd/csrc),
evaluated on the CPU."""

import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CLANG = "/opt/rocm/llvm/bin/clang++"


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    if not os.path.exists(CLANG):
        pytest.skip("no C++ compiler")
    d = tmp_path_factory.mktemp("limits")
    (d / "r.cpp").write_text('''
#include "attn_route.hpp"
using namespace tqt;
extern "C" {
int r_first_key(int pos, int window) { return attn_first_key(pos, window); }
}
''')
    subprocess.run([CLANG, "-O2", "-std=c++17", "-fwrapv", "-fPIC", "-shared", "-Wall", "-I" +
                    os.path.join(ROOT, "torq-tile_amd", "csrc"), "-o", str(d / "r.so"), str(d / "r.cpp")],
                   check=True)
    lib = ctypes.CDLL(str(d / "r.so"))
    lib.r_first_key.argtypes = [ctypes.c_int] * 2
    return lib


POSITIONS = [1 - 2 ** 31, -2 ** 30, -70, -2, -1, 0, 1, 63, 64, 99, 2 ** 30 - 1]


@pytest.mark.parametrize("window", [0, 1, 2, 64, 100, 2 ** 30, 2 ** 31 - 2, 2 ** 31 - 1])
def test_first_key_of_a_window(rules, window):
    """Queries before every key (negative positions) beside windows up to the largest."""
    for pos in POSITIONS:
        want = max(pos - window + 1, 0) if window else 0
        assert rules.r_first_key(pos, window) == want, (pos, window)
