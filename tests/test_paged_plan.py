"""Decisions that the paged cache's kernels take on the device (moa-workspace_amd/csrc/moa_paged_plan.h), compiled for the
host with the device's arithmetic (integers wrap)."""
import ctypes as C
import itertools
import random
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


def arrive(plan, counter, order):
    """The parts of `order`, (first, parts) each, arrive at a counter in turn: its new value, and which arrivals were told to join."""
    joins = []
    for i, (first, parts) in enumerate(order):
        share = plan.join_share(first, parts)
        if plan.join_last(counter, share):
            joins.append(i)
        counter = (counter + share) % 2 ** 32
    return counter, joins


@pytest.mark.parametrize("held", [0, 32, 2 ** 32 - 32])
def test_a_split_sequence_is_joined_by_its_last_part(plan, held):
    rng = random.Random(held)
    for parts in range(2, 17):
        for _ in range(40):
            order = [(i == 0, parts) for i in range(parts)]
            rng.shuffle(order)
            after, joins = arrive(plan, held, order)
            assert joins == [parts - 1] and after % plan.join_turn() == 0


def test_counters_heal_after_calls_that_overlapped(plan):
    """Two launches whose parts arrive at one counter in any order: the next launch joins once, by its last part."""
    rng = random.Random(3)
    for _ in range(500):
        both = []
        for parts in (rng.randrange(2, 17), rng.randrange(2, 17)):
            both += [(i == 0, parts) for i in range(parts)]
        rng.shuffle(both)
        counter, _ = arrive(plan, 32 * rng.randrange(2 ** 27), both)
        parts = rng.randrange(2, 17)
        order = [(i == 0, parts) for i in range(parts)]
        rng.shuffle(order)
        assert arrive(plan, counter, order)[1] == [parts - 1]


def test_the_parts_of_split_tiles_fit_their_records(plan):
    """As many records are there as items. The total comes as short as f32 sums can make it: 1031 roundings of 2^-24."""
    plan.chunk_part_units.argtypes, plan.chunk_part_units.restype = [C.c_float, C.c_int], C.c_int
    rng = random.Random(5)
    for _ in range(20000):
        items = rng.choice([1, 2, 3, 5, 64, 270, 512, rng.randrange(1, 600)])
        tiles, units = int(2 ** rng.uniform(0, 24)), int(2 ** rng.uniform(0, 24))
        for n, u in ((tiles, units), (1, units), (items, units), (max(1, items // 2), units)):
            total = n * u
            part = plan.chunk_part_units(total * (1 - 2.0 ** -24) ** 1031, items)
            parts = -(-u // part)
            assert parts == 1 or (n * parts <= items and part * items >= 2 * total), (items, n, u, part)
