"""CPU: how fft_quad_kernel claims its transforms (cyberether_amd/csrc/kernels/fft_quad.hh).  The counter is asked by an ordinary
vector atomic, nothing waits for the answer in front of the passes, and no GPU source writes through the scalar data cache."""
import os
import re
import shutil
import subprocess
import sys

import pytest

from test_tool_rules import ROOT, sources

sys.path.insert(0, os.path.join(ROOT, "tools"))
SCALAR_CACHE_WRITE = re.compile(r"\bs_(?:buffer_|scratch_)?(?:store|atomic)_\w+|\bs_dcache_(?:wb|inv|discard)\w*")


def test_no_gpu_source_writes_through_the_scalar_data_cache():
    found = [(p, m.group(0)) for p, text in sources("cyberether_amd", "integration", "oracle", "tools")
             if (m := SCALAR_CACHE_WRITE.search(text))]
    assert found == []


@pytest.mark.skipif(shutil.which("hipcc") is None and not os.path.exists("/opt/rocm/bin/hipcc"), reason="no hipcc")
def test_the_claim_is_a_vector_atomic_nobody_waits_for_at_once(tmp_path):
    import check_quad_isa
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    out = tmp_path / "quad.s"
    csrc = os.path.join(ROOT, "cyberether_amd", "csrc")
    subprocess.run([hipcc, "--offload-arch=gfx950", "-O3", "-std=c++20", "-ffp-contract=off", "-Xclang", "-target-feature",
                    "-Xclang", "-packed-fp32-ops", "-S", "--cuda-device-only",
                    "-I", os.path.join(csrc, "kernels"), "-I", csrc, "-I", os.path.join(ROOT, "include"),
                    os.path.join(csrc, "kernels", "fft_side.hip"), "-o", str(out)], check=True, capture_output=True)
    r = check_quad_isa.check(out.read_text())
    assert r["scalar_writes"] == [] and r["waits_behind_the_claim"] == [], r
    assert r["vmcnt"] == r["stores_behind_last_piece"] and not r["other_vmem_between"], r
