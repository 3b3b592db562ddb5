"""Wait states around the inline-assembly MFMAs of the gated feed-forward's large tiles (CPU
test: compiles to gfx950 assembly), by the scanners of test_mfma_hazards."""
import shutil
import subprocess
from pathlib import Path

import pytest
from test_mfma_hazards import accumulator_hazards, build_native, hazards


@pytest.mark.skipif(not Path(build_native.HIPCC).exists() and shutil.which("hipcc") is None,
                    reason="hipcc not available")
def test_inline_mfma_operands_have_their_wait_states(tmp_path):
    out = tmp_path / "gated.s"
    cmd = [build_native.HIPCC, *build_native.HIP_FLAGS, "--cuda-device-only", "-S", str(build_native.CSRC / "gated.hip"), "-o", str(out)]
    res = subprocess.run(cmd, capture_output=True, text=True, timeout=600)
    assert res.returncode == 0, res.stderr[-2000:]
    lines = out.read_text().split("\n")
    assert any("v_mfma_f32_16x16x32_bf16" in line for line in lines), "no 16x16x32 MFMA compiled"
    bad = hazards(lines)
    assert not bad, f"{len(bad)} MFMA operand hazards, first: {bad[:3]}"
    bad = accumulator_hazards(lines)
    assert not bad, f"{len(bad)} accumulator hazards after inline MFMAs, first: {bad[:3]}"
