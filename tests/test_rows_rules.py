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
