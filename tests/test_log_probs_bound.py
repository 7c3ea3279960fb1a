"""The bound below which `log_probs` lists no number: the rule restated, over maxima that other warps raise meanwhile."""
from __future__ import annotations

import os
import random
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cpi_b200", "csrc")


def bound(own, counted, top):
    """What a warp takes as its bound from each lane's own reading and the maxima that the lanes count against it."""
    kept = [v for v in own if sum(o > v for o in counted) < top]
    return min(kept) if kept else None          # (None: the lowest number)


def raised(rng, maxima):
    """The maxima a moment later: other warps have met larger numbers of some lanes."""
    return [m + rng.choice((0, 0, 0, rng.randrange(1, 40))) for m in maxima]


@pytest.mark.parametrize("top", [1, 2, 3, 5, 8, 20, 32])
def test_at_least_top_numbers_are_not_below_the_bound(top):
    rng = random.Random(top)
    for _ in range(300):
        maxima = [rng.randrange(100) for _ in range(32)]
        # each lane may read at a moment of its own: what is counted is the snapshot of what the lanes have read
        own = [rng.choice((a, b)) for a, b in zip(maxima, raised(rng, maxima))]
        assert sum(m >= bound(own, own, top) for m in own) >= top


def test_two_readings_are_no_bound():
    """Why there is one reading only: ranks against maxima that have been read again, later, can leave a lane out by its own newer
    number.  The top 2 of (10, 7, 5): the bound has to let 7 through."""
    own, later = [10, 1, 1, 1], [10, 5, 1, 1]
    assert bound(own, later, 2) == 10 and bound(own, own, 2) == 1
    rng = random.Random(0)
    wrong = 0
    for _ in range(300):
        maxima = [rng.randrange(100) for _ in range(32)]
        later = raised(rng, maxima)
        b = bound(maxima, later, 2)
        wrong += b is not None and sum(m >= b for m in later) < 2
    assert wrong > 0


def test_the_kernel_reads_the_maxima_once():
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, "log_probs.cu")).read())
    body = text[text.index("float bound_of("):]
    body = body[:body.index("\n}\n")]
    meets = re.search(r"if \(together\) __syncthreads\(\); else __syncwarp\(\);", body)
    assert len(re.findall(r"\blane_max\b", body[meets.end():])) == 1
    ranks = body[body.index("int before"):]
    assert "snapshot" in ranks and re.search(r"snapshot\[lane\] = v;\s*__syncwarp\(\);", body)
