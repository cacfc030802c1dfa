"""The device code of the FP8 and grouped products: the wait state of loads to LDS, and no register in memory."""
import re
import subprocess
import sys
from pathlib import Path

import pytest

PKG = Path(__file__).resolve().parents[1] / "unified-memory-scheduler_amd"


@pytest.fixture(scope="module")
def lines(tmp_path_factory):
    sys.path.insert(0, str(PKG))
    import build_lib
    out = tmp_path_factory.mktemp("asm") / "product.s"
    cmd = [build_lib.hipcc(), *build_lib.HIP_FLAGS, f"-I{build_lib.HOST}", "-x", "hip", "-S", "--cuda-device-only",
           str(build_lib.CSRC / "vbm_product.hip"), "-o", str(out)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    assert proc.returncode == 0, proc.stderr
    return [line.strip() for line in out.read_text().splitlines()]


def test_loads_to_lds_are_a_wait_state_behind_their_m0_write(lines):
    """A load to LDS takes its address from M0 and needs one wait state behind a scalar write of it."""
    since, loads, bad = 99, 0, []
    for line in lines:
        if not re.match(r"[svgd][a-z0-9]*_|buffer_|flat_|scratch_", line):
            continue
        if "_load_lds_" in line:
            loads += 1
            bad += [line] if since < 1 else []
        nop = re.match(r"s_nop (\d+)", line)
        since = 0 if re.match(r"s_\w+ m0,", line) else since + (int(nop.group(1)) + 1 if nop else 1)
    assert loads > 0
    assert not bad, (len(bad), bad[:3])


def test_lane_masks_are_restored_behind_the_loads_they_are_for(lines):
    """A load that some waves sit out sets the lanes to none and has to set them back at once."""
    for i, line in enumerate(lines):
        if re.match(r"s_mov_b32 exec_hi, s", line):
            assert "_load_lds_" in lines[i + 1] and re.match(r"s_mov_b64 exec, -1", lines[i + 2]), lines[i:i + 3]


def test_no_kernel_keeps_registers_in_memory(lines):
    """Spilled registers would be reloaded through the counter that the kernels' own waits count on."""
    assert not [line for line in lines if line.startswith("scratch_")]
