"""Decisions that the paged cache's kernels take on the device (moa-workspace_amd/csrc/moa_paged_plan.h), compiled for the
host with the device's arithmetic (integers wrap)."""
import ctypes as C
import itertools
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    lib = tmp_path_factory.mktemp("plan") / "paged_plan.so"
    subprocess.run(["g++", "-std=c++17", "-O2", "-fwrapv", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC",
                    f"-I{ROOT / 'moa-workspace_amd' / 'csrc'}", "-o", str(lib), str(ROOT / "tests" / "cpp" / "paged_plan.cpp")], check=True)
    return C.CDLL(str(lib))


ENDS = [-2 ** 31, -2 ** 31 + 1, -2 ** 31 + 4, -2 ** 30, -5, -1, 0, 1, 3, 4, 5, 2 ** 20, 2 ** 30, 2 ** 31 - 4, 2 ** 31 - 1]


@pytest.mark.parametrize("rows,max_rows", [(4, 4), (4, 1), (1, 1), (2 ** 20, 2 ** 20)])
def test_rows_in_range_at_the_ends_of_int32(plan, rows, max_rows):
    """No pair of row starts leads out of the call's rows, nor to more than max_rows of them: also where their difference wraps."""
    for row0, end in itertools.product(ENDS, ENDS):
        want = 0 <= row0 <= end <= rows and end - row0 <= max_rows
        assert bool(plan.rows_in_range(row0, end, rows, max_rows)) == want, (row0, end)
