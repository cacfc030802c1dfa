"""The rule by which the products choose their kernel (host code), and that the GPU tests' calls reach all of them."""
import subprocess
from pathlib import Path

import pytest

import product_cases as P

REPO = Path(__file__).resolve().parents[1]
NAMES = ["few8", "few16", "stream8_4", "stream8_8", "stream16_4", "stream16_8", "tile256x256", "tile256x160", "tile256x128", "tile128x64", "tile64x32"]


@pytest.fixture(scope="module")
def chosen(tmp_path_factory):
    exe = tmp_path_factory.mktemp("rule") / "test_product_rule"
    subprocess.run(["g++", "-O2", "-std=c++17", f"-I{REPO / 'unified-memory-scheduler_amd' / 'csrc'}",
                    str(REPO / "tests" / "cpp" / "test_product_rule.cpp"), "-o", str(exe)], check=True)

    def ask(calls):
        out = subprocess.run([str(exe)], input="".join(" ".join(map(str, c)) + "\n" for c in calls), capture_output=True, text=True, check=True, timeout=60)
        return out.stdout.split()
    return ask


def test_every_case_reaches_the_kernel_it_is_for(chosen):
    cases = list(P.cases())
    got = chosen([(P.KINDS[types], 1, groups * mean, groups, rows, k * (1 if types[0] == P.F8 else 2)) for types, _, groups, mean, rows, k in cases])
    assert got == [c[1].split()[0] for c in cases]


def test_every_kernel_of_every_kind_is_reached(chosen):
    reached = {(P.KINDS[types], name.split()[0]) for types, name, *_ in P.cases()}
    for kind in range(4):
        for name in NAMES:
            assert (kind, name) in reached or (kind == 0 and name in ("tile256x256", "tile256x160")), (kind, name)


@pytest.mark.parametrize("call,kernel", [
    # kind, grouped, rows, groups, weight rows, bytes of k
    ((0, 0, 1, 1, 5760, 2880), "few8"), ((1, 0, 333, 1, 2880, 2880), "tile64x32"), ((1, 0, 4096, 1, 4096, 4096), "tile256x256"),
    ((0, 0, 4096, 1, 4096, 4096), "tile256x128"), ((1, 1, 8, 128, 1536, 2048), "few8"), ((0, 1, 256, 32, 5760, 2880), "stream16_4"),
    ((1, 1, 16384, 128, 1536, 2048), "tile256x256"), ((3, 1, 64, 32, 2880, 5760), "stream8_4"), ((3, 1, 256, 32, 2880, 5760), "stream16_8"),
    ((2, 1, 9102, 64, 2048, 2816), "tile256x160"), ((1, 0, 2048, 1, 2048, 2048), "tile128x64"), ((3, 1, 256, 32, 2880, 8192), "few16"),
])
def test_ordinary_sizes(chosen, call, kernel):
    assert chosen([call]) == [kernel]
