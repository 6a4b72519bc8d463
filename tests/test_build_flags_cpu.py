"""CPU: the commands that compile the three sources without packed FP32 instructions, as make would run them."""
import os
import shlex
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "datr_amd", "csrc")


@pytest.mark.parametrize("source", ["embedding", "distill", "gemm_i8"])
def test_no_packed_fp32(source):
    lines = subprocess.run(["make", "-Bn", "-C", CSRC], check=True, capture_output=True, text=True).stdout.splitlines()
    compiles = [shlex.split(line) for line in lines if f" -c {source}.hip " in line]
    assert len(compiles) == 1
    words = compiles[0]
    at = words.index("-packed-fp32-ops")
    assert words[at - 3:at] == ["-Xclang", "-target-feature", "-Xclang"]
