"""The compiled 4-bit products hold to what the other matrix kernels are held to."""
import os
import re
import shutil
import subprocess

import pytest


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
    import build_native
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    out = tmp_path_factory.mktemp("q4") / "q4.s"
    r = subprocess.run([hipcc, *build_native.CFLAGS, "--cuda-device-only", "-S",
                        str(build_native.CSRC / "q4.hip"), "-o", str(out)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    return out.read_text()


def test_accumulators_never_partially_overlap(assembly):
    """A matrix instruction accumulates in place or into disjoint registers: partially overlapping
    accumulators have given wrong results on this hardware."""
    pat = re.compile(r"v_mfma\w*\s+([av])\[(\d+):(\d+)\],[^,]+,[^,]+,\s*(?:([av])\[(\d+):(\d+)\]|0)")
    found = list(pat.finditer(assembly))
    assert len(found) > 300 and len(found) == len(re.findall(r"^\s*v_mfma", assembly, re.M))
    chained = 0
    for m in found:
        if m[4] != m[1]:
            continue
        chained += 1
        d0, d1, c0, c1 = map(int, (m[2], m[3], m[5], m[6]))
        assert (d0, d1) == (c0, c1) or d0 > c1 or c0 > d1, m[0]
    assert chained > 100
