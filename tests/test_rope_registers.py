"""The rotation and the append keep eight waves a SIMD in flight, which their loads need (CPU; needs hipcc): the
compiler's resource remarks for every instance of rope_rows_kernel, with and without a norm."""

import os
import re
import subprocess

import pytest

import test_asm_loads as A


@pytest.mark.skipif(not os.path.exists(A.HIPCC), reason="no hipcc")
@pytest.mark.parametrize("source,instances", [("rope_kv.hip", 9), ("norm_rope.hip", 9)])
def test_eight_waves(source, instances, tmp_path):
    flags = [x for x in A.FLAGS if x != "-S"] + ["-Rpass-analysis=kernel-resource-usage"]
    r = subprocess.run([A.HIPCC, *flags, "-c", "csrc/" + source, "-o", str(tmp_path / "x.o")], cwd=A.PKG,
                       capture_output=True, text=True, check=True)
    waves, name = {}, None
    for line in r.stderr.splitlines():
        m = re.search(r"Function Name: (\S+)", line)
        name = m.group(1) if m else name
        m = re.search(r"Occupancy \[waves/SIMD\]: (\d+)", line)
        if m and "rope_rows_kernel" in name:
            waves[name] = int(m.group(1))
    assert len(waves) == instances and all(n == 8 for n in waves.values()), waves
