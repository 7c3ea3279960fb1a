"""Which tails a prompt step gives to other blocks, and how they come back when the step fails (no device needed)."""
from __future__ import annotations

import random

import pytest
import torch

from cpi_b200.cache.kv8 import FORMATS, KeptTails, Kv8Cache, Kv8Plan


def plan_of(starts, news, slots):
    return Kv8Plan(starts, news, slots, device="cpu")


def test_the_tails_that_move():
    rng = random.Random(1)
    for _ in range(300):
        n = rng.randint(1, 5)
        starts = [rng.choice([0, 1, 63, 64, 65, 128, rng.randrange(300)]) for _ in range(n)]
        news = [rng.choice([1, 2, 63, 64, 65, rng.randrange(1, 200)]) for _ in range(n)]
        slots = rng.sample(range(9), n)
        plan = plan_of(starts, news, slots)
        # the tail held rows of the open block, and it holds rows of another one when the step is through
        want = [slot for s, m, slot in zip(starts, news, slots) if s % 64 > 0 and (s + m) % 64 > 0 and s // 64 != (s + m) // 64]
        assert (plan.moved is None and not want) or plan.moved.tolist() == want
        assert plan.jobs.numel() == 8 * plan.n_jobs


@pytest.mark.parametrize("layers", [0, 3])
@pytest.mark.parametrize("fmt", sorted(FORMATS))
def test_kept_tails_come_back(fmt, layers):
    """Of one layer's cache and of several layers' in one."""
    front = (layers,) if layers else ()
    codes, scales = torch.zeros(*front, 3, 2, 64, 64).to(FORMATS[fmt]), torch.ones(*front, 3, 2)
    tails = [torch.randn(*front, 4, 2, 64, 64).bfloat16() for _ in range(4)]
    caches = [Kv8Cache(codes, codes, scales, scales, tails[i].clone(), tails[i + 2].clone()) for i in range(2)]
    plan = plan_of([10, 64, 100, 63], [100, 100, 7, 2], [3, 0, 2, 1])
    assert plan.moved.tolist() == [3, 1]
    kept = KeptTails()
    for c in caches:
        kept.keep(c, plan)
        c.k_tail[:] = 7
        c.v_tail[:] = 7
    kept.put_back()
    for i, c in enumerate(caches):
        for got, want in ((c.k_tail, tails[i]), (c.v_tail, tails[i + 2])):
            assert torch.equal(got[..., [1, 3], :, :, :], want[..., [1, 3], :, :, :]) and (got[..., [0, 2], :, :, :] == 7).all()
    caches[0].k_tail[:] = 5                  # (what has been put back is let go of)
    kept.put_back()
    assert (caches[0].k_tail == 5).all()
    kept.keep(caches[0], plan_of([0, 64], [100, 100], [3, 0]))
    kept.put_back()
    assert (caches[0].k_tail == 5).all()
