"""CPU transcription of the launch arithmetic of the 8-bit cache's attention (lastro-rust_amd/csrc/kv8_attn.hip): which
workgroup takes which column tile of which unit (sequence, KV head and split). Over the limits that the entry points
accept, every pair is taken once and the grid is one that can be launched."""
import os
import random

import pytest

SOURCE = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lastro-rust_amd", "csrc",
                           "kv8_attn.hip")).read()
THREADS = 256


def grid(units, tiles):
    return (units if units < 8 else (units + 7) // 8 * 8) * tiles


def place(i, units, tiles):
    """(unit, tile) of workgroup i; a unit that is not there: none."""
    if units < 8:
        return i % units, i // units
    return i // 8 // tiles * 8 + i % 8, i // 8 % tiles


def test_the_transcription_is_the_source():
    for line in ("const long long grid = (units < 8 ? units : (units + 7) / 8 * 8) * a.tiles;",
                 "const int unit = units < 8 ? id % units : id / 8 / a.tiles * 8 + id % 8;",
                 "const int tile = units < 8 ? id / units : id / 8 % a.tiles;",
                 "if (unit >= units) return;"):
        assert line in SOURCE, line


@pytest.mark.parametrize("tiles", [1, 2, 3, 7, 8, 9, 250])
def test_every_tile_of_every_unit_is_taken_once(tiles):
    for units in list(range(1, 34)) + [64, 255, 256, 1000]:
        got = [p for p in (place(i, units, tiles) for i in range(grid(units, tiles))) if p[0] < units]
        assert sorted(got) == [(u, t) for u in range(units) for t in range(tiles)], units


def test_grids_of_all_that_is_accepted_can_be_launched():
    """A grid has fewer than 2^32 threads. 64 query heads on one KV head and 2^20 positions are 2^21 tiles of one unit."""
    rng = random.Random(1)
    shapes = [(1, 64, 1 << 20), (2, 32, 1 << 20), (7, 18, 1 << 20), (9, 15, 994205), (9, 14, 1 << 20)]
    for _ in range(20000):
        heads = int(2 ** rng.uniform(0, 20))  # KV heads of all sequences
        group = rng.randint(1, 64)
        most = (1 << 27) // (heads * group)
        if most:
            shapes.append((heads, group, min(1 << 20, max(1, int(2 ** rng.uniform(0, 27)) % most + 1))))
    for heads, group, n in shapes:
        cols = group * n
        assert heads * cols <= 1 << 27 and n <= 1 << 20
        width = 16 if cols <= 16 else 32
        tiles = -(-cols // width)
        # splits are added only where a unit of each of 1024 workgroups is not there without them
        for units in (heads, max(heads, 1024 // tiles)):
            assert grid(units, tiles) * THREADS < 1 << 32, (heads, group, n)
