"""Distances of the vector instructions that the kernels of the serving operators issue as inline asm,
which the compiler's hazard recognizer does not look into (CPU only; hipcc cross-compiles). Planted
cases pin the checker."""
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "mini-infer-llama.cpp_amd")

sys.path.insert(0, PKG)
import check_dpp_hazards as chk  # noqa: E402

MFMA = "\tv_mfma_f32_32x32x16_f16 v[0:15], v[20:23], v[24:27], v[0:15]\n"
ASM = "\t;;#ASMSTART\n%s\t;;#ASMEND\n"
MIX = ASM % "\tv_fma_mix_f32 v40, -v41, 1.0, v3 op_sel_hi:[1,0,0]\n"
SWAP = ASM % "\tv_permlane32_swap_b32 v50, v51\n"
NOP_SWAP = ASM % "\ts_nop 1\n\tv_permlane32_swap_b32 v50, v51\n"


@pytest.mark.parametrize("body,found", [
    (MFMA + MIX, 1), (MFMA + "\ts_nop 15\n" + MIX, 1), (MFMA + "\ts_nop 15\n\ts_nop 2\n" + MIX, 0),
    (MFMA + "\tv_add_f32_e32 v3, v60, v61\n" + MIX, 0),                  # written again in between
    (MFMA.replace("v[0:15]", "v[4:19]") + MIX, 0),                        # another register
    ("\tv_exp_f32_e32 v3, v1\n" + MIX, 1), ("\tv_exp_f32_e32 v3, v1\n\ts_nop 0\n" + MIX, 0),
    ("\tv_mov_b32_e32 v51, v50\n" + SWAP, 1), ("\tv_mov_b32_e32 v50, v9\n\ts_nop 0\n" + SWAP, 1),
    ("\tv_mov_b32_e32 v51, v50\n" + NOP_SWAP, 0),
    (MFMA.replace("v[0:15]", "v[36:51]") + "\tv_mov_b32_e32 v50, v9\n" + NOP_SWAP, 1),
    (MFMA + "\tv_fma_mix_f32 v40, -v41, 1.0, v3 op_sel_hi:[1,0,0]\n", 0),  # the compiler's own: its business
    (MFMA + "\ts_cbranch_scc1 .L1\n\ts_nop 15\n\ts_nop 15\n.L1:\n" + MIX, 1),
])
def test_planted(tmp_path, body, found):
    path = tmp_path / "k.s"
    path.write_text("kernel:\n" + body + "\ts_endpgm\n")
    out = []
    for name, items in chk.parse_functions(str(path)).items():
        out += chk.check_asm_function(name, items)
    assert len(out) == found


@pytest.mark.skipif(shutil.which("make") is None or not os.path.exists("/opt/rocm/bin/hipcc"),
                    reason="needs make and hipcc")
def test_generated_kernels():
    subprocess.run(["make", "-C", PKG, "asm"], check=True, capture_output=True, timeout=1200)
    asm = [os.path.join(PKG, "_build", f + ".s") for f in ("tree", "tree_wide", "kv8", "logits")]
    n = bad = 0
    for path in asm:
        for name, items in chk.parse_functions(path).items():
            n += sum(1 for it in items if isinstance(it, chk.Inst) and it.asm)
            bad += len(chk.check_function(name, items)) + len(chk.check_asm_function(name, items))
    assert bad == 0
    assert n > 500  # the multiply-adds and swaps were found
