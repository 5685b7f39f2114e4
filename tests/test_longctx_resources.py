"""Registers of the packed attention and position bias kernels (CPU:
hipcc cross-compiles), with the flags they are built with."""

import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(
    os.path.abspath(__file__))), "dynamic_load_balance_distributeddnn_amd",
    "ops", "csrc")
HIPCC = shutil.which("hipcc")


@pytest.mark.skipif(HIPCC is None, reason="hipcc not on PATH")
@pytest.mark.parametrize("src,most", [
    # the attention kernels fill the registers: a few values that only the
    # masked tiles or the ends use may be put aside, no accumulator (a
    # 32 x 32 one is 64 bytes a lane)
    ("packed_attn_fwd.hip", 60), ("packed_attn_bwd.hip", 60),
    ("relbias.hip", 0)])
def test_scratch(src, most, tmp_path):
    out = subprocess.run(
        [HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
         "-Rpass-analysis=kernel-resource-usage", "-c",
         os.path.join(CSRC, src), "-o", str(tmp_path / "k.o")],
        capture_output=True, text=True, timeout=600)
    assert out.returncode == 0, out.stderr[-2000:]
    found = re.findall(r"Function Name: (\S+).*?ScratchSize "
                       r"\[bytes/lane\]:\s*(\d+).*?LDS Size "
                       r"\[bytes/block\]:\s*(\d+)", out.stderr, re.S)
    assert found, "expected resource remarks"
    assert not [x for x in found if int(x[1]) > most], found
    # two workgroups a CU
    assert not [x for x in found if int(x[2]) > 160 * 1024 // 2], found
