"""Log probabilities of given tokens: rows of many batches with few alternatives, and numbers at the edges, against plain 64-bit
arithmetic."""
from __future__ import annotations

import math

import pytest
import torch

from cpi_b200.csrc import lib as K

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("top", [2, 3, 5, 8])
@pytest.mark.parametrize("rows,vocab", [(700, 40001), (64, 202048), (3, 300003)])
def test_the_best_of_rows_of_many_batches(rows, vocab, top, dtype):
    """Every batch that raises the bound does so while other warps raise the maxima: no number above it may be lost.  Alternatives are
    the row's own numbers, so they are equal, not near."""
    g = torch.Generator(device=DEV).manual_seed(vocab + top)
    x = (torch.randn(rows, vocab, generator=g, device=DEV) * 4).to(dtype)
    ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top].int()
    targets = ids.long()[:, -1:].contiguous()
    for _ in range(20):
        got = K.log_probs(x, targets, top=top)
        assert torch.equal(got.top_ids, ids)
        assert torch.equal(got.top_logprobs[:, -1], got.logprob[:, 0])


def all_nan(got, r):
    return bool(got.logprob[r].isnan().all() and got.entropy[r].isnan() and got.top_logprobs[r].isnan().all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab,cover", [(33, 0), (3001, 0), (3001, 900), (40003, 5000), (151643, 0), (151643, 20000), (202048, 30000)])
def test_a_nan_anywhere_in_a_row(vocab, cover, dtype):
    """At the ends of rows that begin and end beside 16 bytes, in the middle, in any block's share, alone or among masked numbers
    (`cover` of them to either side): the row's probabilities are NaN, the best tokens those of its numbers."""
    places = [0, 1, vocab // 9, vocab // 3, vocab // 2 + 1, vocab - 1000 if vocab > 2000 else 5, vocab - 2, vocab - 1]
    g = torch.Generator(device=DEV).manual_seed(vocab)
    x = (torch.randn(len(places) + 1, vocab, generator=g, device=DEV) * 3).to(dtype)
    for r, at in enumerate(places):
        if cover:
            x[r, max(0, at - cover):at + cover] = -math.inf
        x[r, at] = math.nan
    targets = torch.full((len(places) + 1, 2), vocab // 2, dtype=torch.int32, device=DEV)
    got = K.log_probs(x, targets, top=4)
    ids = torch.sort(x.nan_to_num(-math.inf, neginf=-math.inf), dim=-1, descending=True, stable=True).indices[:, :4].int()
    assert torch.equal(got.top_ids, ids)
    for r, at in enumerate(places):
        assert all_nan(got, r), f"NaN at {at}"
    assert got.logprob[-1].isfinite().all() and got.entropy[-1].isfinite() and got.top_logprobs[-1].isfinite().all()
    bare = K.log_probs(x, targets)
    assert bare.logprob[:-1].isnan().all() and bare.entropy[:-1].isnan().all() and bare.logprob[-1].isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_short_rows_with_nan_and_infinities(dtype):
    nan, inf = math.nan, math.inf
    x = torch.tensor([[nan, nan, 1.0], [1.0, nan, -inf], [-inf, -inf, nan], [inf, 1.0, inf], [inf, -inf, 2.0], [nan, inf, -inf], [0.0, 0.0, -inf]],
                     device=DEV).to(dtype)
    got = K.log_probs(x, torch.zeros(7, dtype=torch.int32, device=DEV), top=3)
    for r in range(6):
        assert all_nan(got, r), f"row {r}"
    assert got.top_ids.tolist() == [[2, -1, -1], [0, 2, -1], [0, 1, -1], [0, 2, 1], [0, 2, 1], [1, 2, -1], [0, 1, 2]]
    assert abs(float(got.entropy[6]) - math.log(2)) < 1e-6 and abs(float(got.logprob[6]) + math.log(2)) < 1e-6


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [5, 2999, 70001])
@pytest.mark.parametrize("big", [0.9e38, 1.1e38, 1.5e38, 3e38])
def test_numbers_near_the_types_largest(big, vocab, dtype):
    """Distances beyond float32 are as good as infinite: nothing but the largest counts."""
    x = torch.full((5, vocab), -math.inf, device=DEV)
    x[0, 3] = big
    x[1, 3], x[1, vocab - 1] = big, big
    x[2, :], x[2, 3] = -big, big
    x[3, :], x[3, 3], x[3, 4] = 0.0, big, -math.inf
    x[4, :], x[4, 3] = -3e38, -big
    x = x.to(dtype)
    got = K.log_probs(x, torch.tensor([[3, 0]] * 5, dtype=torch.int32, device=DEV), top=2)
    ties = [1, 2, 1, 1, 1 if big < 3e38 else vocab]
    for r, n in enumerate(ties):
        assert abs(float(got.entropy[r]) - math.log(n)) < 1e-5, f"row {r}"
        assert abs(float(got.logprob[r, 0]) + math.log(n)) < 1e-5, f"row {r}"
    want = torch.log_softmax(x.double(), -1)[:, 0]
    for r in range(4):                   # (a distance of more than float32's largest is -inf)
        w = float(want[r])
        assert float(got.logprob[r, 1]) == (-math.inf if w < -3.4028235e38 else pytest.approx(w, rel=1e-6))
