"""Distances of the vector instructions that the paged attention kernels issue as inline asm (CPU only;
hipcc cross-compiles). The scan itself is pinned by tests/test_asm_hazards.py."""
import os
import shutil
import subprocess
import sys

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mini-infer-llama.cpp_amd")

sys.path.insert(0, PKG)
import check_dpp_hazards as chk  # noqa: E402


@pytest.mark.skipif(shutil.which("make") is None or not os.path.exists("/opt/rocm/bin/hipcc"),
                    reason="needs make and hipcc")
def test_generated_kernels():
    subprocess.run(["make", "-C", PKG, "asm"], check=True, capture_output=True, timeout=1200)
    n = bad = 0
    uniform = {}
    for name, items in chk.parse_functions(os.path.join(PKG, "_build", "paged_attn.s")).items():
        n += sum(1 for it in items if isinstance(it, chk.Inst) and it.asm)
        bad += len(chk.check_function(name, items)) + len(chk.check_asm_function(name, items))
        uniform[name] = sum(1 for it in items if isinstance(it, chk.Inst) and it.op == "v_readfirstlane_b32")
    assert bad == 0
    assert n > 500
    # descriptors are in scalar registers: where the compiler takes one for a lane's own it loads through a
    # loop, four to six more of these for each load (378 in a kernel instead of 39)
    kernels = {k: v for k, v in uniform.items() if "paged_" in k}
    assert len(kernels) == 18 and min(kernels.values()) > 5 and max(kernels.values()) < 100, kernels
