"""The cut of a packed batch into tiles (csrc/kf_attention.hip, ``locate``), restated: every row in exactly one tile, of its own sequence or of
none; and the refusals of kf_attention_starts."""

import random

import pytest

from kronfluence_amd import _native as nat

ROWS = 128


def tile(offsets, total, slot):
    """(first row of the sequence, its rows, its visible tokens, row of the tile in it), or None"""
    sequences = len(offsets) - 1
    offset = lambda s: total if s > sequences else min(max(offsets[s], 0), total)
    first_slot = lambda s: offset(s) // ROWS + s
    front = offset(0)
    if slot < front // ROWS or slot == total // ROWS + sequences + 1:
        row0 = min(slot, front // ROWS) * ROWS
        return (0, front, 0, row0) if row0 < front else None
    lo, hi = 0, sequences
    while lo < hi:
        mid = (lo + hi + 1) // 2
        lo, hi = (mid, hi) if first_slot(mid) <= slot else (lo, mid - 1)
    begin, rows = offset(lo), max(offset(lo + 1) - offset(lo), 0)
    t = slot - first_slot(lo)
    return (begin, rows, 0 if lo == sequences else rows, t * ROWS) if 0 <= t < -(-rows // ROWS) else None


@pytest.mark.parametrize("seed", range(40))
def test_every_row_of_a_packed_batch_is_in_one_tile(seed):
    rng = random.Random(seed)
    total = rng.choice([1, 2, 127, 128, 129, 300, 1000, 1024])
    offsets = sorted(rng.choice([0, total, rng.randint(0, total), min(total, ROWS * rng.randint(0, 8))]) for _ in range(rng.choice([2, 3, 4, 9, 60])))
    owner = [None] * total
    for slot in range(total // ROWS + len(offsets) - 1 + 2):
        found = tile(offsets, total, slot)
        if found is not None:
            begin, rows, visible, row0 = found
            for row in range(begin + row0, begin + min(rows, row0 + ROWS)):
                assert owner[row] is None, (offsets, total, row)
                owner[row] = (begin, visible)
    for row in range(total):
        inside = [(a, b - a) for a, b in zip(offsets, offsets[1:]) if a <= row < b]
        assert owner[row] is not None and (owner[row] == inside[0] if inside else owner[row][1] == 0), (offsets, total, row)


def test_starts_refuse():
    call = lambda starts=16, offsets=16, dtype=nat.KF_I32, sequences=3, rows=10: nat.lib().kf_attention_starts(starts, offsets, dtype, sequences, rows, None)
    assert call(dtype=nat.KF_F32) == -2
    for bad in (dict(starts=None), dict(offsets=None), dict(sequences=-1), dict(rows=-1), dict(rows=1 << 31)):
        assert call(**bad) == -1, bad
