"""What test_mfma_waits.py checks is the code that ships: its compiler flags are the Makefile's, but for warnings and where the output goes."""
import os
import shlex
import shutil
import subprocess

import pytest

from test_mfma_waits import FLAGS, ROOT

CSRC = os.path.join(ROOT, "buffer-x_amd", "csrc")


def _flags_of_make(source):
    said = subprocess.run(["make", "-n", "-W", source, f"_obj/{source[:-4]}.o", "HIPCC=hipcc"], cwd=CSRC, check=True, capture_output=True, text=True).stdout
    words = shlex.split([line for line in said.splitlines() if line.startswith("hipcc ") and source in line][-1])[1:]
    at = words.index("-c")
    assert words[at + 1] == source and words[at + 2] == "-o"
    return [w for w in words[:at] + words[at + 4:] if not w.startswith("-W")]


@pytest.mark.skipif(not shutil.which("make"), reason="needs make")
@pytest.mark.parametrize("source", ["k_linear.hip", "k_attn.hip"])
def test_the_checked_code_is_the_shipped_code(source):
    assert _flags_of_make(source) == [f for f in FLAGS if f not in ("--cuda-device-only", "-S")]


@pytest.mark.skipif(not shutil.which("make"), reason="needs make")
def test_no_packed_f32_in_the_dense_operators():
    for source in ("k_linear.hip", "k_rope.hip", "k_attn.hip"):
        flags = _flags_of_make(source)
        assert any(flags[i:i + 4] == ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"] for i in range(len(flags)))
