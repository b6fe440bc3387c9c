"""What the 4-bit K/V cache's kernels need of the compiler, looked for in its listing."""
import re
import shutil
import subprocess

import pytest

from conftest import ROOT

HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


def registers(operand):
    m = re.fullmatch(r"([va])\[(\d+):(\d+)\]", operand) or re.fullmatch(r"([va])(\d+)", operand)
    return {(m[1], i) for i in range(int(m[2]), int(m[m.lastindex]) + 1)} if m else set()


@pytest.mark.skipif(not shutil.which(HIPCC), reason="no hipcc here")
def test_fp6_conversions_keep_apart(tmp_path):
    """A conversion of 32 values between float32 and fp6 writes while it still reads: its result lies on none of its sources."""
    out = tmp_path / "kv4.s"
    flags = ["--offload-arch=gfx950", "-O3", "-std=c++17", f"-I{ROOT / 'include'}", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-mllvm",
             "-amdgpu-mfma-vgpr-form=1", "--cuda-device-only", "-S"]
    subprocess.run([HIPCC, *flags, "-o", str(out), str(ROOT / "l3m_amd" / "csrc" / "kv4.hip")], check=True, capture_output=True, timeout=600)
    seen = 0
    for line in out.read_text().splitlines():
        m = re.match(r"\s+v_cvt_scalef32_(?:2xpk16_fp6_f32|pk32_f32_fp6)\S*\s+(.*)", line)
        if m:
            to, *sources = (registers(x.strip()) for x in m[1].split(";")[0].split(","))
            seen += 1
            assert to and sources[0] and not any(to & x for x in sources), line
    assert seen >= 100
