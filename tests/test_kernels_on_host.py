"""The paged attention (with and without trees), the plan, the kept rows and the norm with its gradient on the CPU: the
kernels' own sources and launches (tests/host_hip.hpp, tests/host_kernels.py), on arrays whose every neighbour is a page
that may not be touched, in an order of waves, lanes and workgroups that is drawn anew each time, against the plain forms."""

import os
import subprocess
import sys

import pytest

import host_kernels as K

pytestmark = pytest.mark.skipif(not os.path.exists(K.CLANG), reason="no C++ compiler")


@pytest.fixture(scope="module")
def library(tmp_path_factory):
    return K.build(str(tmp_path_factory.mktemp("host")))


@pytest.mark.parametrize("suite,seed", [("attention", 1), ("attention", 2), ("spans", 1), ("plan", 1), ("plan", 2),
                                        ("keep", 1), ("keep", 2), ("norm", 1), ("norm", 2)])
def test_random_calls(library, suite, seed):
    r = subprocess.run([sys.executable, os.path.join(K.ROOT, "tests", "host_kernels.py"), library, suite, str(seed)],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.endswith("whole\n"), (r.returncode, r.stdout[-600:], r.stderr[-1500:])
