"""The packed attention kernels' loads to LDS, in the assembly that hipcc
makes of them (CPU: it cross-compiles)."""

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
@pytest.mark.parametrize("src", ["packed_attn_fwd.hip",
                                 "packed_attn_bwd.hip"])
def test_a_load_waits_for_what_it_reads(src, tmp_path):
    """A vector memory access must not follow the vector instruction that
    wrote its scalar address (a readlane: a spilled address coming back) by
    less than five wait states, and the compiler counts none for code
    written as assembly.  So the block itself copies the address by a
    scalar instruction, for which the hardware waits, and that copy is the
    wait state between the write of M0 and the load."""
    out = tmp_path / "k.s"
    run = subprocess.run(
        [HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
         "-S", "--cuda-device-only", os.path.join(CSRC, src), "-o",
         str(out)], capture_output=True, text=True, timeout=600)
    assert run.returncode == 0, run.stderr[-2000:]
    text = out.read_text()
    blocks = re.findall(r";;#ASMSTART(.*?);;#ASMEND", text, re.S)
    loads = [b for b in blocks if "global_load_lds" in b]
    assert len(loads) > 100
    assert text.count("global_load_lds") == len(loads)
    for block in loads:
        lines = [line.split(";")[0].strip() for line in block.splitlines()]
        m0, copy, load = [line for line in lines if line]
        assert re.fullmatch(r"s_mov_b32 m0, s\d+", m0), block
        base = re.fullmatch(r"s_mov_b64 (s\[\d+:\d+\]), \S+", copy)
        assert base, block
        assert load.startswith("global_load_lds_dword")
        assert load.endswith(", " + base[1]), block
