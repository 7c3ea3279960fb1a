"""Requests for scores that cannot be answered are refused before anything runs (no device needed)."""
from __future__ import annotations

from types import SimpleNamespace

import pytest

from cpi_b200.api import Model
from cpi_b200.cache.manager import CacheError
from cpi_b200.csrc import lib as K
from cpi_b200.engine.generate import GenerationRequest
from cpi_b200.engine.score import score_sequence
from test_generation_loop import FakeEngine, gen


def fake(vocab):
    e = FakeEngine(vocab=vocab)
    e.spec = SimpleNamespace(vocab_size=vocab)
    return e


@pytest.mark.parametrize("vocab,logprobs", [(50, 33), (50, -1), (20, 21), (20, 32), (50, 1000)])
def test_generation_refuses_alternatives_that_there_are_not(vocab, logprobs):
    e = fake(vocab)
    with pytest.raises(ValueError, match="request 1: logprobs"):
        gen(e, max_batch=4).generate([GenerationRequest([1, 2], 2), GenerationRequest([3], 2, logprobs=logprobs)])
    assert not e.acquired and not e.steps


class Untouched:
    """An engine of which nothing but its sizes is looked at."""
    max_step_tokens, device = 8, "cpu"

    def __init__(self, vocab=50, room=True):
        self.spec, self.slots, self.asked = SimpleNamespace(vocab_size=vocab), [], []
        self.cache = SimpleNamespace(check_room=self.check_room)

    def check_room(self, pieces):
        self.asked += pieces
        raise CacheError("no room")

    def acquire_slot(self):
        self.slots.append(5)
        return 5

    def release_slot(self, slot):
        self.slots.remove(slot)

    def step(self, entries):
        raise AssertionError("a step was run")


@pytest.mark.parametrize("vocab,top", [(50, 33), (50, -1), (20, 21)])
def test_scores_refuse_alternatives_that_there_are_not(vocab, top):
    e = Untouched(vocab)
    with pytest.raises(ValueError, match="alternatives"):
        score_sequence(e, [1, 2, 3], top)
    assert not e.asked


def test_a_text_that_does_not_fit_is_refused_before_its_first_piece():
    e = Untouched()
    with pytest.raises(CacheError, match="no room"):
        score_sequence(e, [1] * 21)
    assert e.asked == [([5], [8]), ([5], [8]), ([5], [4])] and not e.slots


@pytest.mark.parametrize("texts", [[[1, 2], [3]], [[1, 2], [3, 50]], [[1, 2], [-1, 3]]])
def test_no_text_is_scored_if_one_cannot_be(texts):
    m = Model.__new__(Model)
    m.engine = Untouched()
    with pytest.raises(ValueError):
        m.score(texts)
    with pytest.raises(ValueError):
        m.score([[1, 2]], top=33)
    assert not m.engine.asked


def test_the_most_is_what_the_kernel_lists():
    assert K.log_probs_most() == 32
