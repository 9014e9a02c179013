"""Spilled registers of the unquantised operators' kernels, from the
compiler's own report.  The 256-row tiles' few are stored before their loop and
were measured to be free; the tokens kernels' are of fp32 rows with 17 to 32
picks."""
import os
import re
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "system-lab_amd"))

from smoe import build  # noqa: E402


@pytest.mark.parametrize("name,most", [("smoe_tokens", 8), ("smoe_linear", 0), ("smoe_linear_mm", 5),
                                       ("smoe_linear_rows", 0)])
def test_spilled_registers(name, most):
    src = os.path.join(ROOT, "system-lab_amd", "csrc", name + ".hip")
    flags = [f for f in build.HIP_FLAGS if not f.startswith("-W")]
    r = subprocess.run([build.HIPCC, *flags, "--cuda-device-only", "-Rpass-analysis=kernel-resource-usage", "-c", src,
                        "-o", os.devnull], check=True, capture_output=True, text=True, timeout=900)
    names = re.findall(r"Function Name: (\S+)", r.stderr)
    spills = [int(n) for n in re.findall(r"VGPRs Spill: (\d+)", r.stderr)]
    assert len(names) == len(spills) > 0
    assert max(spills) <= most, [(n, s) for n, s in zip(names, spills) if s > most]
