"""The device code of the layer for a few tokens: wait states that the loads to LDS need, and no register in memory. The loads are inline assembly,
into which the compiler does not count."""
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
    out = tmp_path_factory.mktemp("asm") / "few.s"
    cmd = [build_lib.hipcc(), *build_lib.HIP_FLAGS, f"-I{build_lib.HOST}", "-x", "hip", "-S", "--cuda-device-only",
           str(build_lib.CSRC / "vbm_moe_few.hip"), "-o", str(out)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    assert proc.returncode == 0, proc.stderr
    return [line.strip() for line in out.read_text().splitlines()]


def instructions(lines):
    """(operation, operands, wait states) one after the other; None where a function begins."""
    for line in lines:
        if line.endswith(":") and line.startswith("_Z"):
            yield None
        if re.match(r"[svgd][a-z0-9]*_|buffer_|flat_|scratch_", line):
            op, _, rest = line.partition(" ")
            nop = re.match(r"s_nop (\d+)", line)
            yield op, [a.strip().split(" ")[0] for a in rest.split(",")], int(nop.group(1)) + 1 if nop else 1


def scalars(operand):
    pair = re.match(r"s\[(\d+):(\d+)\]$", operand)
    if pair:
        return set(range(int(pair.group(1)), int(pair.group(2)) + 1))
    one = re.match(r"s(\d+)$", operand)
    return {int(one.group(1))} if one else set()


def test_loads_are_five_wait_states_behind_vector_writes_of_their_scalar_base(lines):
    recent, loads, bad = [], 0, []
    for i in instructions(lines):
        if i is None:
            recent = []
            continue
        op, operands, states = i
        if "_load_lds_" in op:
            loads += 1
            used, apart = set().union(*map(scalars, operands)), 0
            for written, n in reversed(recent):
                if apart < 5 and written & used:
                    bad.append((op, operands, apart))
                apart += n
        recent = recent[-15:] + [(scalars(operands[0]) if op.startswith("v_") else set(), states)]
    assert loads > 0 and not bad, (len(bad), bad[:3])


def test_loads_are_a_wait_state_behind_their_m0_write(lines):
    since, loads, bad = 99, 0, []
    for i in instructions(lines):
        if i is None:
            continue
        op, operands, states = i
        if "_load_lds_" in op:
            loads += 1
            bad += [operands] if since < 1 else []
        since = 0 if op.startswith("s_mov") and operands[0] == "m0" else since + states
    assert loads > 0 and not bad, (len(bad), bad[:3])


def test_no_kernel_keeps_registers_in_memory(lines):
    """Spilled registers would be reloaded through the counter that the kernels' own waits count on."""
    assert not [line for line in lines if line.startswith("scratch_")]
