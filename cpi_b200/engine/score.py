"""Scores of given tokens: a sequence is run as a prompt, and every position's logits say how probable the next token was.

The logits of a piece (float32 [tokens, vocab]) live in one buffer of the engine's, which keeps the size that its largest step
needed; pieces are cut so that it stays below LOGIT_BYTES.  Each
piece's rows go through one launch of `log_probs`; nothing else of them is kept.  (The reference scores nothing: it prints the
largest logits after a prompt, src/engine/llama4_cuda_engine.cu:623-674.)
"""
from __future__ import annotations

from typing import Sequence

import torch

from ..csrc import lib as K
from .engine import StepEntry

LOGIT_BYTES = 1 << 30


def most_alternatives(engine) -> int:
    return min(K.log_probs_most(), engine.spec.vocab_size)


def check_scored(engine, tokens: Sequence[int], top: int = 0) -> list:
    """The tokens as a list, if they and `top` can be scored; a ValueError if not."""
    tokens, vocab = [int(t) for t in tokens], engine.spec.vocab_size
    if len(tokens) < 2:
        raise ValueError("a sequence to score has two tokens or more: the first is given, the others are scored")
    if min(tokens) < 0 or max(tokens) >= vocab:
        raise ValueError(f"a token id lies outside the vocabulary of {vocab}")
    if not 0 <= top <= most_alternatives(engine):
        raise ValueError(f"scores list up to {most_alternatives(engine)} alternatives, not {top}")
    return tokens


def score_sequence(engine, tokens: Sequence[int], top: int = 0) -> "K.LogProbs":
    """Of tokens t_0 .. t_{n-1} (n >= 2) the log probabilities of t_1 .. t_{n-1} given what precedes each, the entropy of each
    distribution and its `top` best tokens: a LogProbs of n - 1 rows on the device."""
    tokens = check_scored(engine, tokens, top)
    n = len(tokens) - 1
    piece = max(1, min(engine.max_step_tokens, LOGIT_BYTES // (4 * engine.spec.vocab_size)))
    slot = engine.acquire_slot()
    parts = []
    try:
        # all pieces fit, or none runs
        engine.cache.check_room([([slot], [min(piece, n - a)]) for a in range(0, n, piece)])
        targets = torch.tensor(tokens[1:], dtype=torch.int32, device=engine.device)
        for a in range(0, n, piece):
            b = min(n, a + piece)
            logits = engine.step([StepEntry(slot, tokens[a:b], range(b - a))])
            parts.append(K.log_probs(logits, targets[a:b], top=top))
        engine.check_device_errors()
    finally:
        engine.release_slot(slot)
    if len(parts) == 1:
        return parts[0]
    return K.LogProbs(*(None if c[0] is None else torch.cat(c) for c in zip(*parts)))
