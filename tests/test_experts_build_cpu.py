"""Build-time guard for the expert tiles (CPU, no GPU needed): their LDS-DMA is written in inline asm,
whose scalar operands the compiler cannot pad for, and the sweep of a K loop must not spill."""
import os
import re
import shutil
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
SRC = os.path.join(ROOT, "smoothquant-mixedprecision_amd", "csrc", "sqmp_experts.hip")


@pytest.mark.skipif(shutil.which("hipcc") is None and not os.path.exists("/opt/rocm/bin/hipcc"),
                    reason="hipcc not available")
def test_expert_tiles_build(tmp_path):
    import build_ext
    flags = [f for f in build_ext.CFLAGS if f != "-fPIC"]
    asm = str(tmp_path / "experts.s")
    r = subprocess.run([build_ext.HIPCC, *flags, "--cuda-device-only", "-S", SRC, "-o", asm,
                        "-Rpass-analysis=kernel-resource-usage"], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
    # no asm memory instruction reads a scalar register that a vector instruction wrote less than
    # five wait states before
    sys.path.insert(0, os.path.join(ROOT, "tools"))
    import check_asm_sgpr_hazard as H
    assert H.main(asm) == 0
    text = open(asm).read()
    assert not re.search(r"v_pk_(add|mul|fma)_f32", text)     # built without packed fp32
    blocks = re.split(r"remark: [^\n]*Function Name: ", r.stderr)
    seen = 0
    for b in blocks[1:]:
        if "expert_tiles_kernel" not in b.split()[0]:
            continue
        seen += 1
        assert int(re.search(r"VGPRs Spill: (\d+)", b).group(1)) == 0, b.split()[0]
        assert int(re.search(r"Occupancy \[waves/SIMD\]: (\d+)", b).group(1)) >= 2
    assert seen == 16        # fp16 / bf16 x groups of 64 / 32 x gated or not x 128 / 256 rows
