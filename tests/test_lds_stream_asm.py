"""The device code of every kernel that streams weights to LDS with a scalar base: a load needs five wait states behind a vector instruction that writes
its base. The loads are inline assembly, into which the compiler does not count, so its output is checked: back from each load along every way
that leads to it, branches and loops included."""
import re
import subprocess
import sys
from pathlib import Path

import pytest

PKG = Path(__file__).resolve().parents[1] / "unified-memory-scheduler_amd"
STATES = 5


def registers(operand):
    """The scalar registers that an operand names."""
    pair = re.match(r"s\[(\d+):(\d+)\]$", operand)
    if pair:
        return {f"s{i}" for i in range(int(pair.group(1)), int(pair.group(2)) + 1)}
    if operand == "vcc":
        return {"vcc_lo", "vcc_hi"}
    return {operand} if re.match(r"s\d+$|vcc_lo$|vcc_hi$", operand) else set()


class Instruction:
    def __init__(self, line):
        op, _, rest = re.sub(r"\s*(;|//).*", "", line).replace("\t", " ").partition(" ")
        self.line, self.op = line, op
        self.operands = [a.strip().split(" ")[0] for a in re.split(r",(?![^\[]*\])", rest)]
        nop = re.match(r"s_nop (\d+)", line)
        self.states = int(nop.group(1)) + 1 if nop else 1
        # (a carry or a scale flag is a vector instruction's second result)
        results = self.operands[:2] if re.match(r"v_\w+_co_|v_div_scale|v_mad_[iu]64", op) else self.operands[:1]
        self.written = set().union(*map(registers, results)) if op.startswith("v_") else set()
        self.load = "_load_lds_" in op
        self.base = set().union(*map(registers, self.operands)) if self.load else set()


def functions(text):
    """Each function's instructions, and for each of them those that can come right before it."""
    for body in re.split(r"^_Z\S*:.*$", text, flags=re.M)[1:]:
        code, labels, jumps = [], {}, []
        for line in (raw.strip() for raw in body.splitlines()):
            label = re.match(r"(\.L\w+):", line)
            if label:
                labels[label.group(1)] = len(code)
            if line.startswith(".Lfunc_end"):
                break
            if re.match(r"[svgd][a-z0-9]*_|buffer_|flat_|scratch_", line):
                code.append(Instruction(line))
                if code[-1].op.startswith(("s_branch", "s_cbranch")):
                    jumps.append((len(code) - 1, code[-1].operands[-1]))
        before = [[i - 1] if i and code[i - 1].op not in ("s_branch", "s_endpgm", "s_setpc_b64") else [] for i in range(len(code))]
        for at, label in jumps:
            if labels[label] < len(code):
                before[labels[label]].append(at)
        yield code, before


def too_close(code, before, at):
    """A vector instruction that writes the base of load `at` fewer than STATES wait states ahead of it, or None."""
    ways, seen = [(p, 0) for p in before[at]], {}
    while ways:
        i, apart = ways.pop()
        if apart >= STATES or seen.get(i, STATES) <= apart:
            continue
        seen[i] = apart
        if code[i].written & code[at].base:
            return code[i].line, apart
        ways += [(p, apart + code[i].states) for p in before[i]]
    return None


def check(text):
    """(loads with a scalar base, those that come too early)."""
    loads, bad = 0, []
    for code, before in functions(text):
        for at, i in enumerate(code):
            if i.load and i.base:
                loads += 1
                near = too_close(code, before, at)
                bad += [(i.line, *near)] if near else []
    return loads, bad


def test_the_check_follows_branches_and_counts_wait_states():
    body = """_Z1kv:                                  ; @_Z1kv
	v_readfirstlane_b32 s5, v1
	s_nop {n}
	s_branch .LBB0_2
.LBB0_1:
	s_nop 9
.LBB0_2:
	s_mov_b32 m0, s2
	s_nop 0
	global_load_lds_dwordx4 v0, s[4:5]
	{write}
	s_cbranch_scc1 .LBB0_2
	s_endpgm
.Lfunc_end0:
"""
    count = lambda **kw: [len(b) if isinstance(b, list) else b for b in check(body.format(**kw))]  # noqa: E731
    assert count(n=1, write="s_nop 9") == [1, 0] and count(n=0, write="s_nop 9") == [1, 1]
    assert count(n=5, write="v_cmp_eq_u32_e64 s[4:5], v0, v1") == [1, 1] and count(n=5, write="v_add_co_u32_e64 v1, s[4:5], v0, v1") == [1, 1]
    assert count(n=5, write="v_readlane_b32 s6, v0, 1") == [1, 0]


SOURCES = sorted(p.name for p in (PKG / "csrc").glob("*.hip") if "vbm_lds_stream.hpp" in p.read_text())


@pytest.fixture(scope="module")
def device_code(tmp_path_factory):
    """name -> the device code of a source (all are compiled at once)."""
    sys.path.insert(0, str(PKG))
    import build_lib
    out = {name: tmp_path_factory.mktemp("asm") / (name + ".s") for name in SOURCES}
    runs = {name: subprocess.Popen([build_lib.hipcc(), *build_lib.HIP_FLAGS, f"-I{build_lib.HOST}", "-x", "hip", "-S", "--cuda-device-only",
                                    str(build_lib.CSRC / name), "-o", str(path)], stderr=subprocess.PIPE, text=True) for name, path in out.items()}
    for run in runs.values():
        _, err = run.communicate()
        assert run.returncode == 0, err
    return {name: path.read_text() for name, path in out.items()}


@pytest.mark.parametrize("source", SOURCES)
def test_loads_are_five_wait_states_behind_vector_writes_of_their_base(device_code, source):
    loads, bad = check(device_code[source])
    assert loads > 100 and not bad, (len(bad), bad[:3])
