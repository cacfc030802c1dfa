"""The strips' calls reach the kernels that they are for, with more token tiles in a group than a strip's eight and a remainder."""
import subprocess
from pathlib import Path

import i8_strip_cases as S

REPO = Path(__file__).resolve().parents[1]
STRIP = 8


def test_every_case_reaches_its_kernel_and_fills_strips(tmp_path):
    exe = tmp_path / "rule"
    subprocess.run(["g++", "-O2", "-std=c++17", f"-I{REPO / 'unified-memory-scheduler_amd' / 'csrc'}", str(REPO / "tests" / "cpp" / "test_i8_product_rule.cpp"),
                    "-o", str(exe)], check=True)
    calls = [(1, sum(counts), len(counts), rows, k) for counts, rows, k in S.CASES.values()]
    out = subprocess.run([str(exe)], input="".join(" ".join(map(str, c)) + "\n" for c in calls), capture_output=True, text=True, check=True, timeout=60)
    assert out.stdout.split() == list(S.CASES)
    for name, (counts, rows, _) in S.CASES.items():
        rows_a_tile, tokens_a_tile = map(int, name[4:].split("x"))
        tiles = [-(-(-(-n // 16)) // (tokens_a_tile // 16)) for n in counts]
        assert rows > rows_a_tile and any(n > STRIP and n % STRIP for n in tiles), (name, tiles)
        assert any(tiles[:next(i for i, n in enumerate(tiles) if n > STRIP)]) or any(n > STRIP for n in tiles[1:]), name   # (not the first group alone)
