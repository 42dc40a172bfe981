"""Every tile of lines of sequences of unlike rows is one workgroup's, and no workgroup has another: the kernels' own rule, compiled for the CPU."""
import collections
import ctypes as C
import os
import random
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
LINES = 128


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    path = str(tmp_path_factory.mktemp("attend_tiles") / "attend_tiles.so")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-o", path, os.path.join(HERE, "attend_tiles.cpp")])
    lib = C.CDLL(path)
    lib.numbers.restype = C.c_long

    def tiles(starts, rows, group):
        n = len(starts) - 1
        count = lib.numbers(rows, group, LINES, n)
        which, tile = (C.c_int * count)(), (C.c_long * count)()
        lib.tiles((C.c_int * (n + 1))(*starts), n, rows, group, LINES, C.c_long(count), which, tile)
        return list(zip(which, tile))

    return tiles


def check(rule, starts, rows, group):
    clamped = [min(max(s, 0), rows) for s in starts]
    had = collections.Counter((s, t) for s, t in rule(starts, rows, group) if s >= 0)
    assert all(t >= 0 for _, t in had)
    wanted = {(s, t) for s in range(len(starts) - 1) for t in range(-(-(clamped[s + 1] - clamped[s]) * group // LINES))}
    assert {k: had[k] for k in wanted} == dict.fromkeys(wanted, 1)
    # beyond a sequence's lines: at most one number, which finds nothing to do
    assert all(count == 1 for count in had.values())


@pytest.mark.parametrize("starts, rows, group", [
    ([64, 464], 464, 4), ([32, 33], 40, 4), ([31, 33], 40, 4), ([128, 128, 328], 328, 1), ([1000, 1000, 1000], 1000, 8), ([1000, 1500], 1500, 8),
    ([0, 400], 400, 4), ([0, 0, 0, 129, 129, 500], 700, 1), ([-5, 4, 8, 1000], 48, 4), ([2000, 2100, 2 ** 31 - 1], 1500, 3), ([5, 5], 5, 64),
])
def test_every_tile_is_taken_once(rule, starts, rows, group):
    check(rule, starts, rows, group)


def test_every_tile_of_drawn_batches_is_taken_once(rule):
    rng = random.Random(5)
    for _ in range(400):
        starts = [rng.choice((0, rng.randint(0, 40), rng.randint(100, 900)))]
        for _ in range(rng.randint(1, 9)):
            starts.append(starts[-1] + rng.choice((0, 1, rng.randint(2, 40), rng.randint(41, 700))))
        check(rule, starts, starts[-1] + rng.choice((0, 7)), rng.choice((1, 2, 3, 4, 5, 8, 14, 40, 128, 200)))


def test_starts_that_decrease_name_no_tile_that_is_not_there(rule):
    for starts in ([40, 30, 20, 10], [2 ** 31 - 1, -(2 ** 31), 0, 5], [900, 0, 500, 2]):
        assert all(s == -1 or (0 <= s < 3 and t >= 0) for s, t in rule(starts, 1000, 4))
