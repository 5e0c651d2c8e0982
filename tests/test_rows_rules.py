"""The launch rules of the operators between two attention blocks on the CPU."""
import shutil
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("g++ is not installed")
    exe = tmp_path_factory.mktemp("rules") / "rows_rules_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    str(HERE / "rows_rules_check.cpp"), "-o", str(exe)], check=True)

    def evaluate(name, *args):
        out = subprocess.run([str(exe)], input=" ".join(map(str, (name, *args))), capture_output=True, text=True, check=True)
        return int(out.stdout)

    return evaluate


@pytest.mark.parametrize("rows", [1, 2, 1000, 2 ** 21 - 1, 2 ** 21, 2 ** 21 + 1, 3 * 2 ** 20, 2 ** 22 - 1, 2 ** 22])
def test_workgroups_of_long_rows(rule, rows):
    """Threads along x stay below 2^32, along y few; every row has a workgroup, and at most one launch's worth has none."""
    columns = rule("long_row_columns", rows)
    lines = -(-rows // columns)
    assert columns * 1024 < 2 ** 32 and lines <= 65535
    assert rows <= columns * lines < rows + columns


@pytest.mark.parametrize("tokens,rows,side", [
    (1, 2560, 0), (64, 2560, 0), (300, 1000, 0), (830, 704, 0), (830, 833, 64), (64, 12288, 64), (16, 10241, 64), (1024, 2560, 64),
    (256, 12288, 128), (1800, 1801, 128), (4003, 1536, 128), (3601, 3587, 256), (4096, 12288, 256), (8192, 8192, 256)])
def test_tiles_of_the_projection(rule, tokens, rows, side):
    assert rule("linear8_tile", tokens, rows, 1536, 256) == side
    assert rule("linear8_tile", tokens, rows, 1 << 24, 256) == 0


def test_tiles_of_the_projection_at_the_limits(rule):
    for tokens in (1, 2 ** 22):
        for rows in (1, 2 ** 20):
            side = rule("linear8_tile", tokens, rows, 65536, 256)
            assert side in (0, 64, 128, 256) and (side or tokens * rows < 2 ** 20)
