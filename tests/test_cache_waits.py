"""Bounded waits of the cache attention kernels, on the CPU.

Each lane of a warp polls and reads the clock by itself, so a wait that runs out
may do so for some lanes and not for others. What follows a wait is the whole
warp's (mma.sync, shuffles, ldmatrix), so the lanes have to agree on the outcome:
`mbar_wait_warp` and `ck_wait` vote, `mbar_wait_bounded` does not and belongs in
code that one lane runs."""

from __future__ import annotations

import random
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "fast-moss-diarization_b200" / "csrc"


def _one_lane_only(source: str, call: str):
    """(line, whether a block opened for a single lane encloses it) of each call."""
    text = re.sub(r"//[^\n]*", lambda m: " " * len(m.group()), source)
    found, blocks, start = [], [], 0
    for m in re.finditer(r"[{};]|" + call + r"\s*\(", text):
        if m.group() == "{":
            blocks.append(text[start:m.start()])
        elif m.group() == "}":
            blocks.pop()
        if m.group() in "{};":
            start = m.end()
        else:
            single = any(re.search(r"if \((lane|tid) == \d+\)\s*$", b) for b in blocks)
            found.append((text.count("\n", 0, m.start()) + 1, single))
    return found


def test_the_search_tells_one_lane_from_a_warp():
    src = "void f() {\n  if (lane == 0) {\n    for (;;) w(a);\n  }\n  if (!w(b)) x();\n}\n"
    assert _one_lane_only(src, "w") == [(3, True), (5, False)]


@pytest.mark.parametrize("name", ["fmd_cache_decode.cu", "fmd_cache_chunk.cu"])
def test_waits_of_a_whole_warp_vote(name):
    calls = _one_lane_only((CSRC / name).read_text(), "mbar_wait_bounded")
    assert calls and all(single for _, single in calls), calls


def _lanes(rng, limit):
    """Whether each lane's polls see the barrier complete before its own clock runs out."""
    done = rng.randrange(2 * limit)
    return [done <= limit + rng.randrange(-2, 3) for _ in range(32)]


def test_a_vote_leaves_no_warp_divided():
    """The model behind the rule: lanes with clock readings of their own divide a
    warp where they decide alone; one vote never does."""
    rng = random.Random(0)
    divided = 0
    for _ in range(2000):
        lanes = _lanes(rng, 50)
        divided += len(set(lanes)) == 2
        assert len({all(lanes) for _ in lanes}) == 1
    assert divided > 0
