"""The dense operators' matrix kernels, checked without a GPU: nothing reads a matrix instruction's result before it is there, on any path
(tools/mfma_waits.py).  A mask test of two branches behind the scores' products once made f32 attention over heads of 128 read one of them early."""
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tools"))
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-ffp-contract=off", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "--cuda-device-only", "-S"]


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")
@pytest.mark.parametrize("source,kernels", [("k_linear.hip", 60), ("k_attn.hip", 24)])
def test_results_are_waited_for(tmp_path, source, kernels):
    import mfma_waits
    asm = str(tmp_path / "kernels.s")
    subprocess.run([HIPCC] + FLAGS + [os.path.join(ROOT, "buffer-x_amd", "csrc", source), "-o", asm], check=True, stderr=subprocess.DEVNULL, timeout=1200)
    seen = {n: f for n, f in mfma_waits.functions(asm).items() if any(op.startswith("v_mfma") for op, _ in f[0])}
    assert len(seen) >= kernels
    assert {n: e for n, e in ((n, mfma_waits.early(*f)) for n, f in seen.items()) if e} == {}


def test_the_shorter_path_counts(tmp_path):
    """the checker itself: six states on the taken branch, twelve on the other one"""
    import mfma_waits
    text = "f:\n\tv_mfma_f32_32x32x16_bf16 a[0:15], v[2:5], v[6:9], a[0:15]\n\ts_cbranch_vccnz .LBB0_2\n" + "\ts_mov_b32 s0, 0\n" * 10 + \
           ".LBB0_2:\n\ts_nop %d\n\tv_accvgpr_read_b32 v0, a15\n\ts_endpgm\n.Lfunc_end0:\n"
    for nop, bad in ((4, [(0, 13, 6, 12)]), (9, [(0, 13, 11, 12)]), (10, [])):
        path = tmp_path / "f.s"
        path.write_text(text % nop)
        assert mfma_waits.early(*mfma_waits.functions(str(path))["f"]) == bad
