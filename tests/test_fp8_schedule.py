"""The order of LDS copies and reads in the fp8 product on tiles of 256 x 256, on the CPU.

Its waves meet once a stage, so an LDS read by one wave and a copy by another are ordered only by the barriers
between them.  A stage's steps are written down here with the numbers that csrc/k_fp8big.hip gives them, and
every read has to lie before the barrier that the copy into its place follows, and behind the one that the
copy's wait precedes."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

SOURCE = Path(__file__).resolve().parents[1] / "strix-halo-int4-gemms_amd" / "csrc" / "k_fp8big.hip"
STEPS = 34


def _number(text, name, otherwise):
    found = re.search(rf"\b{name}\s*=\s*(\d+)", text)
    return int(found.group(1)) if found else otherwise


@pytest.fixture(scope="module")
def numbers():
    text = SOURCE.read_text()
    later = re.search(r"step >= (\d+) && step % 2 == 0\) piece\(later, slot,", text)
    soon = re.search(r"step < (\d+) && step % 2 == 0\) piece\(soon, slot \^ 1, 4 \+ step / 2\)", text)
    assert later and soon, "the copies of a stage are written another way: write this schedule anew"
    return {"read": _number(text, "kRead", 23), "scales": _number(text, "kCopyScales", 8),
            "slots": _number(text, "kScaleSlots", 2), "later": int(later.group(1)),
            "soon": range(0, min(int(soon.group(1)), 8), 2)}


def _events(n, stages, row_scales):
    """(place, time, kind) of a wave: places are ("rows", slot) and ("scales", slot), times (stage, step), the copy
    of a stage's barrier wait ends at it."""
    reads, copies = [], []
    for i in range(stages):
        for step in range(0, 32, 4):  # row tiles of a and a's scales, two ahead
            ahead = step // 4 >= 6
            reads.append((("rows", (i + ahead) % 2), (i, step), i + ahead))
            reads.append((("scales", (i + ahead) % n["slots"]), (i, step), i + ahead))
        for step in range(24, 28):  # b's of the next stage
            reads.append((("rows", (i + 1) % 2), (i, step), i + 1))
        if row_scales:
            reads += [(("scales", i % n["slots"]), (i, step), i) for step in range(2, STEPS)]
        else:
            reads.append((("scales", (i + 1) % n["slots"]), (i, 24), i + 1))
        copies += [(("rows", i % 2), (i, step), i + 2) for step in range(n["later"], 32, 2)]
        copies += [(("rows", (i + 1) % 2), (i, step), i + 1) for step in n["soon"]]
        copies.append((("scales", (i + 1) % n["slots"]), (i, n["scales"]), i + 1))
    return reads, copies


def _epoch(n, at):
    """Barriers that lie before a time: a stage's is behind step `read`."""
    return at[0] + (at[1] > n["read"])


def _races(n, row_scales, stages=12):
    reads, copies = _events(n, stages, row_scales)
    found = []
    for place, when, wanted in reads:
        for where, issued, brought in copies:
            if where != place:
                continue
            first = _epoch(n, issued)  # the copy ends with the wait at the next barrier
            if _epoch(n, when) == first:
                found.append((place, when, wanted, issued, brought))
    return found


@pytest.mark.parametrize("row_scales", [False, True])
def test_no_copy_meets_a_read(numbers, row_scales):
    assert _races(numbers, row_scales) == []


@pytest.mark.parametrize("row_scales", [False, True])
def test_reads_find_their_stage(numbers, row_scales):
    """What a read finds is the last copy into its place, and that is the stage it wants."""
    reads, copies = _events(numbers, 12, row_scales)
    for place, when, wanted in reads:
        before = [c for c in copies if c[0] == place and _epoch(numbers, c[1]) < _epoch(numbers, when)]
        if before and wanted > 1:  # the first stages are brought before the loop
            assert max(before, key=lambda c: c[1])[2] == wanted


def test_two_slots_of_scales_would_meet(numbers):
    assert _races({**numbers, "slots": 2}, True) and not _races({**numbers, "slots": 2}, False)
