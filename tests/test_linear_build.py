"""Compile-time invariants of the product kernels that their speed depends on (CPU: hipcc only).

The tile kernels keep up to 128 sums and two sets of operands per lane in
registers: a spill, or a kernel that drops below its two waves per SIMD, slows
them several times with no test of values noticing."""
import re
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT / "home-seek_amd"))


@pytest.mark.skipif(shutil.which("/opt/rocm/bin/hipcc") is None, reason="hipcc not present")
def test_linear_kernels_no_scratch_two_waves_per_simd(tmp_path):
    import _build
    src = _build.CSRC / "hsmoe_linear.hip"
    cmd = [_build.HIPCC, *_build.HIP_FLAGS, *_build.SOURCE_FLAGS["hsmoe_linear"], "--offload-device-only",
           "-Rpass-analysis=kernel-resource-usage", "-c", str(src), "-o", str(tmp_path / "linear.o")]
    res = subprocess.run(cmd, capture_output=True, text=True, timeout=600)
    assert res.returncode == 0, res.stderr[-2000:]
    found = {}
    for block in re.split(r"remark: [^\n]*Function Name: ", res.stderr)[1:]:
        found[block.split()[0]] = (int(re.search(r"ScratchSize \[bytes/lane\]: (\d+)", block).group(1)),
                                   int(re.search(r"Occupancy \[waves/SIMD\]: (\d+)", block).group(1)))
    kinds = ("linear_kernel", "linear_narrow_kernel", "linear_grad_input_kernel", "linear_grad_weight_kernel")
    for kind in kinds:
        kernels = {n: v for n, v in found.items() if kind in n}
        assert kernels, (kind, list(found))
        bad = {n: v for n, v in kernels.items() if v[0] != 0}
        assert not bad, f"kernels with scratch: {bad}"
    big = {n: v for n, v in found.items() if "ILi256ELi256" in n}
    assert big and all(occ >= 2 for _, occ in big.values()), big
