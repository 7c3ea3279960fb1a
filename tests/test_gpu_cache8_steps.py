"""Steps of models whose attention layers keep their keys and values in 8 bits: the error word, steps that fail."""
from __future__ import annotations

import pytest
import torch

import tiny
from cpi_b200.csrc import lib as K
from cpi_b200.engine import StepEntry
from test_gpu_cache8_engine import engine, vocab

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("word", [1, 2, 3, 4, 5])
def test_the_error_word_says_which_kind_it_was(word):
    """A wait that ran out in a kernel on CTA pairs is not an index outside of the cache."""
    e = engine("dense", "int8")
    e.check_device_errors()
    K.device_error_flags(torch.device(DEV))[0] = word
    with pytest.raises(RuntimeError, match="outside of the cache" if word == K.INDEX_OUTSIDE else "gave up waiting"):
        e.check_device_errors()
    e.check_device_errors()


def steps(e, seqs, cuts, fail=None, monkeypatch=None, end=True):
    """Logits of each step of `cuts` (tokens per sequence and step) for sequences side by side.  `fail` = (step, call, name):
    the call-th call of that kernel raises once, in that step, which is then run again."""
    slots = [e.acquire_slot() for _ in seqs]
    at, got = [0] * len(seqs), []
    for n, cut in enumerate(cuts):
        entries = [StepEntry(s, t[a:a + c], range(c)) for s, t, a, c in zip(slots, seqs, at, cut) if c]
        if fail is not None and fail[0] == n:
            whole, calls = getattr(K, fail[2]), []

            def failing(*a, **k):
                calls.append(1)
                if len(calls) == fail[1]:
                    raise RuntimeError("out of memory, say")
                return whole(*a, **k)

            with monkeypatch.context() as m:
                m.setattr(K, fail[2], failing)
                with pytest.raises(RuntimeError, match="out of memory, say"):
                    e.step([StepEntry(s, t[a:a + c], range(c)) for s, t, a, c in zip(slots, seqs, at, fail[3]) if c])
            assert [e.length(s) for s in slots] == at
        got.append(e.step(entries).clone())
        at = [a + c for a, c in zip(at, cut)]
    e.check_device_errors()
    for s in slots:
        e.release_slot(s)
    e.cache.check_consistency()
    return got


@pytest.mark.parametrize("held", ["int8", "e4m3"])
@pytest.mark.parametrize("call,name", [(1, "attention_prefill_kv8"), (3, "kv8_stage"), (4, "attention_prefill_kv8")])
@pytest.mark.parametrize("again", [[(70, 20, 64), (1, 1, 1)], [(30, 20, 10), (40, 50, 300)], [(1, 1, 1), (90, 1, 1)]])
def test_a_step_that_failed_is_run_again(again, call, name, held, monkeypatch):
    """A prompt's later piece, which leaves the open block of one sequence for another one, fails in some layer: the same piece, a
    smaller one or a single token after it give the bits that they give without the failure."""
    e = engine("dense", held)
    seqs = [tiny.random_tokens(n, vocab("dense"), n) for n in (300, 290, 500)]
    first = (100, 70, 130)
    want = steps(e, seqs, [first] + again)
    got = steps(e, seqs, [first] + again, fail=(1, call, name, (70, 20, 64)), monkeypatch=monkeypatch)
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_two_failures_in_a_row(monkeypatch):
    e = engine("dense", "int8")
    seqs = [tiny.random_tokens(300, vocab("dense"), 5)]
    want = steps(e, seqs, [(100,), (100,)])
    slot = e.acquire_slot()
    e.step([StepEntry(slot, seqs[0][:100], [])])
    for call in (4, 2):
        whole, calls = K.attention_prefill_kv8, []

        def failing(*a, **k):
            calls.append(1)
            if len(calls) == call:
                raise MemoryError
            return whole(*a, **k)

        with monkeypatch.context() as m:
            m.setattr(K, "attention_prefill_kv8", failing)
            with pytest.raises(MemoryError):
                e.step([StepEntry(slot, seqs[0][100:200], range(100))])
    assert torch.equal(want[1], e.step([StepEntry(slot, seqs[0][100:200], range(100))]))
    e.release_slot(slot)


@pytest.mark.parametrize("name", ["dense", "beside", "turned"])
def test_a_steps_plans_are_there_before_its_first_kernel(name, monkeypatch):
    """Their tables are read by kernels that do not wait for the kernel in front first: no layer makes one."""
    e = engine(name, "int8")
    windows = {(g.req.window_kind, g.req.window_size, g.req.keep_first) for g in e.cache.groups if g.kv8 is not None}
    whole, seen = e.model.run, []

    def run(batch, cache):
        seen.append(set(batch.plans))
        made = dict(batch.plans)
        logits = whole(batch, cache)
        assert batch.plans.keys() == made.keys()
        return logits

    monkeypatch.setattr(e.model, "run", run)
    steps(e, [tiny.random_tokens(200, vocab(name), 1)], [(100,), (50,), (50,)])
    assert seen == [windows] * 3 and windows
