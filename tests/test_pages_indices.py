"""Index arithmetic of the paged cache's kernels, transcribed: every row of a packed batch is some tile's, exactly once and
whatever the lengths; starts of any value lead to no row outside the batch; every block of a tile has one wave and split;
the positions that a lane holds of a product of scores are those that lie side by side in V."""
import numpy as np
import pytest

import pages_util as pu


def first_tile(starts, tokens, g, s, w):
    return min(max(starts[s], 0), tokens) * g // w + s


def find(starts, tokens, g, y, w, seqs):
    """64 candidates at a time, as the lanes of a wave."""
    lo, n = 0, seqs
    while n > 1:
        step = (n + 63) // 64
        hits = [lane for lane in range(64) if lane * step < n and first_tile(starts, tokens, g, lo + lane * step, w) <= y]
        x = max(hits) if hits else 0
        lo += x * step
        n = min(step, n - x * step)
    return lo


def tile(starts, tokens, g, y, w, seqs):
    """(sequence, its place in the batch, first row, rows) of tile y, or None."""
    s = find(starts, tokens, g, y, w, seqs)
    lo = min(max(starts[s], 0), tokens)
    n = min(max(starts[s + 1], lo), tokens) - lo
    at = -(-n * g // w) - 1 - (y - first_tile(starts, tokens, g, s, w))  # the last ones first
    return (s, lo, at * w, n * g) if n >= 1 and 0 <= at < -(-n * g // w) else None


def tiles(tokens, g, w, seqs):
    return tokens * g // w + seqs


@pytest.mark.parametrize("w", [16, 128])
@pytest.mark.parametrize("seqs", [1, 2, 7, 64, 65, 130])
def test_every_row_has_one_tile(w, seqs):
    rng = np.random.default_rng(seqs + w)
    for i in range(6):
        g = int(rng.choice([1, 3, 5, 16, 64]))
        new = rng.choice([0, 0, 1, 1, 2, 3, 17, 43, 128, 300] if i % 2 else [0, 1], seqs)
        before = int(rng.choice([0, 0, 13]))  # rows that belong to no sequence
        starts = (before + np.concatenate([[0], np.cumsum(new)])).tolist()
        tokens = starts[-1] + int(rng.integers(0, 40))
        seen = np.zeros((tokens, g), int)
        for y in range(tiles(tokens, g, w, seqs)):
            t = tile(starts, tokens, g, y, w, seqs)
            if t is None:
                continue
            s, lo, row0, rows = t
            assert starts[s] == lo and rows == new[s] * g
            r = np.arange(row0, min(row0 + w, rows))
            np.add.at(seen, (lo + r // g, r % g), 1)
        assert (seen[before:starts[-1]] == 1).all() and not seen[:before].any() and not seen[starts[-1]:].any()


@pytest.mark.parametrize("w", [16, 128])
def test_broken_starts_lead_to_no_row_outside(w):
    rng = np.random.default_rng(w)
    for _ in range(300):
        seqs, tokens, g = int(rng.integers(1, 200)), int(rng.integers(1, 400)), int(rng.choice([1, 3, 64]))
        starts = rng.choice([-2 ** 31, -7, 0, 1, 2, 5, tokens // 2, tokens - 1, tokens, tokens + 1, 2 ** 31 - 1], seqs + 1).tolist()
        for y in rng.integers(0, tiles(tokens, g, w, seqs), 20):
            t = tile(starts, tokens, g, int(y), w, seqs)
            if t:
                s, lo, row0, rows = t
                assert 0 <= s < seqs and 0 <= lo + row0 // g and lo + (min(row0 + w, rows) - 1) // g < tokens


def test_every_block_has_one_wave_of_few_rows():
    for blocks in list(range(0, 70)) + [333]:
        for splits in (1, 2, 5, 64):
            used = max(1, min(splits, (blocks + 3) // 4))
            got = [b for split in range(used) for wave in range(4)
                   for b in range(split * 4 + wave, blocks, splits * 4)]
            assert sorted(got) == list(range(blocks))


def test_every_stage_has_one_split_of_many_rows():
    for stage in (1, 2):
        for blocks in list(range(0, 70)) + [333]:
            for splits in (1, 2, 5, 64):
                stages, used = -(-blocks // stage), max(1, min(splits, (blocks + 7) // 8))
                got = [x for split in range(used) for x in range(split, stages, used)]
                assert sorted(got) == list(range(stages)) and used <= max(1, stages)


@pytest.mark.parametrize("d", [64, 128])
def test_lanes_hold_what_lies_side_by_side_in_v(d):
    for group in range(4):  # of 16 lanes, few rows: rows 4 group + i of product z
        held = [16 * ((4 * group + i) // 8) + 8 * z + (4 * group + i) % 8 for z in range(2) for i in range(4)]
        assert [pu.v_place(t, 5, d) for t in held] == [(group * d + 5) * 8 + j for j in range(8)]
    for half in range(2):  # of 32 lanes, many rows: register r of a product
        for s2 in range(2):
            held = [8 * (r // 4) + 4 * half + r % 4 for r in range(8 * s2, 8 * s2 + 8)]
            assert [pu.v_place(t, 5, d) for t in held] == [((2 * s2 + half) * d + 5) * 8 + j for j in range(8)]
    for k in range(d // 16):  # a step of 32x32x16 is 1 KB of K
        got = [pu.k_place(lane % 32, 16 * k + 8 * (lane // 32)) for lane in range(64)]
        assert got == [k * 512 + lane * 8 for lane in range(64)]
