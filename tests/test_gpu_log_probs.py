"""Log probabilities of given tokens, entropies and the best alternatives, against plain 64-bit arithmetic."""
from __future__ import annotations

import math

import pytest
import torch

from cpi_b200.csrc import lib as K

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def plain(x, targets, top):
    x = x.double()
    lp = torch.log_softmax(x, -1)
    chosen = lp.gather(-1, targets.long().view(x.shape[0], -1)).view(targets.shape)
    p = lp.exp()
    entropy = -(p * torch.where(p > 0, lp, torch.zeros_like(lp))).sum(-1)
    values, ids = torch.sort(x, dim=-1, descending=True, stable=True)
    return chosen, entropy, lp.gather(-1, ids[:, :top]), ids[:, :top].int()


def compare(x, targets, top):
    got = K.log_probs(x, targets, top=top)
    torch.cuda.synchronize()
    chosen, entropy, best, ids = plain(x, targets, top)
    # A thread adds up to vocab / 512 terms in float32, each off by 2^-22 (the exponential) and 2^-24 per addition: Z and
    # the entropy's sum are off by (2^-22 + n 2^-24) relative, n = vocab / 512 + 32 for the merges; differences x - m are
    # rounded by 2^-24 of their size.
    n = x.shape[1] / 512 + 32
    rel = 2.0 ** -22 + n * 2.0 ** -24
    near = lambda a, b, extra=0.0: bool(((a.double() - b).abs() <= rel * (1 + extra) + 2.0 ** -22 * b.abs())[b.isfinite()].all())       # noqa: E731
    same = lambda a, b: torch.equal(a.double()[~b.isfinite()], b[~b.isfinite()])       # noqa: E731
    assert near(got.logprob, chosen) and same(got.logprob, chosen)
    assert near(got.entropy, entropy, extra=1 + entropy)
    if top:
        assert torch.equal(got.top_ids, ids)
        assert near(got.top_logprobs, best) and same(got.top_logprobs, best)
    else:
        assert got.top_logprobs is None and got.top_ids is None


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 2, 0), (3, 5, 5), (2, 31, 20), (1, 500, 32), (7, 1001, 1), (1, 32000, 5), (5, 32003, 32),
                                            (1, 202048, 20), (8, 202048, 20), (40, 65537, 7), (300, 4099, 3), (1000, 777, 0), (1300, 129, 32), (1300, 5001, 20), (1184, 16384, 1)])
def test_random_rows(dtype, rows, vocab, top):
    g = torch.Generator(device=DEV).manual_seed(vocab + rows)
    x = (torch.randn(rows, vocab, generator=g, device=DEV) * 4).to(dtype)
    compare(x, torch.randint(0, vocab, (rows,), generator=g, device=DEV, dtype=torch.int32), top)


@pytest.mark.parametrize("offset", [0, 1, 2, 3, 5])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_alignment(dtype, offset):
    g = torch.Generator(device=DEV).manual_seed(offset)
    store = (torch.randn(6, 5003, generator=g, device=DEV) * 3).to(dtype)
    x = store[1:, offset:offset + 4217]
    targets = torch.randint(0, 4217, (5, 3), generator=g, device=DEV)       # int64, several per row
    compare(x, targets, 9)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [130, 40000])
def test_ties_and_order(dtype, vocab):
    """Equal numbers come lowest id first; rows that rise, fall, are all alike or hold a few values only."""
    i = torch.arange(vocab, device=DEV).float()
    rows = torch.stack([torch.zeros(vocab, device=DEV), i / vocab * 9, -i / vocab * 9, (i % 3), (i % 7 == 6).float() * 5, (i * 7919 % vocab) / vocab])
    compare(rows.to(dtype), torch.tensor([0, vocab - 1, 0, 5, 6, 17], dtype=torch.int32, device=DEV), 32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [64, 30001])
def test_masks(dtype, vocab):
    g = torch.Generator(device=DEV).manual_seed(1)
    x = (torch.randn(5, vocab, generator=g, device=DEV) * 3).to(dtype)
    low = torch.finfo(dtype).min
    x[0, torch.rand(vocab, generator=g, device=DEV) < 0.7] = -math.inf
    x[1, :] = -math.inf
    x[1, 17] = 2.5                                  # one token left
    x[2, torch.rand(vocab, generator=g, device=DEV) < 0.7] = low
    x[3, :] = low                                   # nothing but the type's lowest value: all alike
    x[4, 20:] = -math.inf                           # fewer tokens than alternatives
    targets = torch.tensor([17, 17, 17, 17, 25], dtype=torch.int32, device=DEV)
    x[0, 17] = x[2, 17] = 1.0
    compare(x, targets, 32)


def test_rows_without_a_distribution():
    x = torch.randn(4, 3000, device=DEV)
    x[0, :] = -math.inf
    x[1, 1234] = math.nan
    x[2, 77] = math.inf
    got = K.log_probs(x, torch.tensor([5, 5, 5, 5], dtype=torch.int32, device=DEV), top=4)
    assert float(got.logprob[0]) == -math.inf and float(got.entropy[0]) == 0.0
    assert got.top_ids[0].tolist() == [0, 1, 2, 3] and (got.top_logprobs[0] == -math.inf).all()
    for r in (1, 2):
        assert got.logprob[r].isnan() and got.entropy[r].isnan() and got.top_logprobs[r].isnan().all()
    assert 1234 not in got.top_ids[1].tolist() and int(got.top_ids[2, 0]) == 77
    assert got.logprob[3].isfinite() and got.entropy[3].isfinite()
    few = torch.full((1, 3), math.nan, device=DEV)
    few[0, 2] = 1.0
    got = K.log_probs(few, torch.zeros(1, dtype=torch.int32, device=DEV), top=3)
    assert got.top_ids[0].tolist() == [2, -1, -1]


def test_targets_that_are_none():
    x = torch.randn(2, 100, device=DEV)
    got = K.log_probs(x, torch.tensor([[-1, -100, 3], [100, 99, 10 ** 6]], device=DEV), top=0).logprob
    want = torch.log_softmax(x.double(), -1)
    assert got[0, :2].tolist() == [0.0, 0.0] and got[1, 0].isnan() and got[1, 2].isnan()
    assert abs(float(got[0, 2] - want[0, 3])) < 1e-5 and abs(float(got[1, 1] - want[1, 99])) < 1e-5


def test_targets_beyond_32_bits():
    """Their low halves would name tokens of the vocabulary."""
    x = torch.randn(2, 100, device=DEV)
    got = K.log_probs(x, torch.tensor([[2 ** 32 + 5, 2 ** 40], [-2 ** 32 + 5, -2 ** 62]], device=DEV), top=0).logprob
    assert got[0].isnan().all() and got[1].tolist() == [0.0, 0.0]


def test_large_logits_and_peaks():
    x = torch.randn(4, 9001, device=DEV) * 1e4
    x[1] = x[1] * 1e-4 + 3e4
    x[2, 5] = 1e30
    x[3] = -1e30
    x[3, 9] = 0.0
    compare(x, torch.tensor([5, 6, 5, 9], dtype=torch.int32, device=DEV), 6)


def test_streams_and_graphs():
    xs = [torch.randn(3, 50001, device=DEV) for _ in range(2)]
    t = torch.tensor([1, 2, 3], dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    K.log_probs(xs[0], t, top=5)
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(K.log_probs(x, t, top=5))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for x, got in zip(xs, outs):
        chosen, _, _, ids = plain(x, t, 5)
        assert torch.equal(got.top_ids, ids) and (got.logprob.double() - chosen).abs().max() < 1e-4


def test_no_rows():
    got = K.log_probs(torch.empty(0, 10, device=DEV), torch.empty(0, dtype=torch.int32, device=DEV), top=2)
    assert got.logprob.shape == (0,) and got.top_ids.shape == (0, 2)
