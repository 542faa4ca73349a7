"""Static checks on the listings of the kernels as the Makefile builds them (no GPU needed: hipcc cross-compiles): none uses
packed fp32 arithmetic, some of whose forms have given wrong results on this hardware, and the hand-scheduled persistent
kernels keep their wait states under those flags (tools/check_mfma_hazard.py)."""
import glob
import os
import re
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "polygon_amd", "csrc")
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


def _flags():
    """CXXFLAGS of the Makefile, its variables filled in."""
    text = open(os.path.join(CSRC, "Makefile")).read()
    var = dict(re.findall(r"^(\w+) \??= (.*)$", text, re.M))
    flags = var["CXXFLAGS"]
    for _ in range(4):
        flags = re.sub(r"\$\((\w+)\)", lambda m: var[m.group(1)], flags)
    return flags.split()


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not available")
@pytest.mark.parametrize("src", sorted(os.path.basename(p) for p in glob.glob(os.path.join(CSRC, "*.hip"))))
def test_listing_as_built(src, tmp_path):
    out = str(tmp_path / (src + ".s"))
    subprocess.run([HIPCC, *_flags(), "--cuda-device-only", "-S", os.path.join(CSRC, src), "-o", out], check=True,
                   stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL, timeout=600)
    assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", open(out).read())
    if src.startswith("pg_persist"):
        r = subprocess.run([sys.executable, os.path.join(ROOT, "tools", "check_mfma_hazard.py"), out], capture_output=True,
                           text=True, timeout=300)
        assert r.returncode == 0 and "0 MFMA hazards" in r.stdout and "0 early touches" in r.stdout, r.stdout[-2000:]
