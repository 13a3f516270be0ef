"""tools/build_variant.sh compiles with the library's own flags."""
import os
import subprocess

import pytest

from conftest import ROOT


def test_variant_builds_take_the_librarys_flags(tmp_path):
    import build_native
    if not list(build_native.BUILD.glob("*.o")):
        pytest.skip("no built objects")
    r = subprocess.run(["bash", "tools/build_variant.sh", str(tmp_path / "v.so"), "dropout.hip",
                        "-DNAME=1"], cwd=ROOT, env={**os.environ, "HIPCC": "echo"},
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    compiled, linked, _ = r.stdout.splitlines()
    assert compiled.startswith(" ".join(build_native.CFLAGS) + " -DNAME=1 -c ")
    assert "-packed-fp32-ops" in compiled and "-shared" in linked
