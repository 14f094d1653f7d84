"""Registers of the linear cross entropy's passes (CPU: hipcc cross-compiles
gfx950 here).  A pass streams chunks through LDS while it multiplies the chunk
before; a spilled value read back in that loop waits for every load in flight.
Two tiles a wave at 256 columns fill the registers, so a few spills remain
there: this keeps them few."""
import os
import re
import shutil
import subprocess
import sys

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ikea-recommender-system_amd")


def test_the_passes_hardly_spill():
    cc = next((c for c in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")) if c and os.path.exists(c)), None)
    if cc is None:
        pytest.skip("hipcc not available")
    sys.path.insert(0, PKG)
    import build
    flags = [f for f in build.FLAGS if f != "-fPIC"]
    r = subprocess.run([cc, *flags, "--cuda-device-only", "-c", "-Rpass-analysis=kernel-resource-usage", "-I", build.CSRC,
                        os.path.join(build.CSRC, "linear_ce.hip"), "-o", os.devnull], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    spills = dict(re.findall(r"Function Name: (\S*k_ce_pass\S*) .*?VGPRs Spill: (\d+)", r.stderr, re.S))
    assert len(spills) == 24
    assert all(int(n) <= 8 for n in spills.values()), spills
