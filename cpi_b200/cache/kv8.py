"""The cache in 8 bits: its tensors, and the pages that a step of several tokens works on.

Positions 64 b .. 64 b + 63 of a sequence are its block b, one page.  A complete block is held as codes of 8 bits with one
power of two as scale per page and key/value head, keys and values each (an element stands for code * scale); the block of
the newest position is held in bfloat16, in the sequence's *tail*, until it is complete.  A query sees the keys and values
of its own block in bfloat16 and those of earlier blocks as held in 8 bits, whatever step brought them: what a position
attends to does not depend on how its sequence was cut into steps.  (Its numbers may by a rounding: other steps project rows by
products of other shapes, and single tokens and prompts round probabilities differently.  Values have to be finite: one that is not
also reaches earlier queries of its sequence within a prompt's key tile.)

  "int8"   scale = the smallest power of two with max |x| <= 127 scale; code = x / scale to the nearest integer
  "e4m3"   max |x| / scale in [128, 256); code = x / scale to the nearest e4m3 number

int8 is finer for numbers of like size; e4m3 keeps the relative precision of small numbers in a block with large ones.
"""
from __future__ import annotations

from typing import NamedTuple

import numpy as np
import torch

BLOCK = 64                       # positions of a block, and of a page
FORMATS = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


class Kv8Cache(NamedTuple):
    """One layer's cache.  Pages are shared by the slots through a page table; tails belong to slots."""
    k: torch.Tensor              # int8 or float8_e4m3fn [pages, kv heads, 64, head_dim]
    v: torch.Tensor
    k_scale: torch.Tensor        # float32 [pages, kv heads], powers of two
    v_scale: torch.Tensor
    k_tail: torch.Tensor         # bfloat16 [slots, kv heads, 64, head_dim]: row p % 64 is position p of the slot's newest block
    v_tail: torch.Tensor


def needed_blocks(start: int, new: int, window_kind: str, window_size: int, keep_first: int) -> list:
    """The blocks that a step of `new` tokens from position `start` reads in 8 bits: those before the last token's own
    that its first token's window, or the kept first positions, reach."""
    low = 0
    if window_kind == "chunk":
        low = start // window_size * window_size
    elif window_kind == "sliding":
        low = max(0, start - window_size + 1)
    keep = keep_first if window_kind == "sliding" else 0
    own = (start + new - 1) // BLOCK
    first = low // BLOCK
    return list(range(min(-(-keep // BLOCK), first))) + list(range(first, own))


class Kv8Plan:
    """Where a step's tokens and the blocks that they see lie among the step's own bfloat16 pages.  Made once per step and
    window (`starts`, `n_new`, `slots` per sequence, as in a StepBatch), used by every layer with that window.

    The pages hold all that the step's sequences see in bfloat16, 4 x kv heads x head size bytes a position, while a layer's
    attention runs.

    Pages 0 .. n_earlier - 1 hold earlier blocks; pages n_earlier .. n_pages - 1 the blocks that the step's tokens fall into,
    sequence after sequence from each one's first new block on.  `exact_table` and `earlier_table` [sequences, width] name
    them per block (-1: none); a kernel that stores rows through a page table stores them through `exact_table` with
    `seq_ids` as the sequences' slots.  `moved`: the slots whose tail the step gives to another block, or None: a caller that may
    have to run the step again keeps those tails (`KeptTails`), as the rows in them are held nowhere else."""

    def __init__(self, starts, n_new, slots, *, window_kind: str = "full", window_size: int = 0, keep_first: int = 0, device="cuda"):
        if not len(starts) == len(n_new) == len(slots) or not len(starts):
            raise ValueError("Kv8Plan: a start, a number of tokens and a slot per sequence")
        if min(n_new) < 1 or min(starts) < 0 or min(slots) < 0:
            raise ValueError("Kv8Plan: sequences bring a token or more, from position 0 on")
        if window_kind not in ("full", "chunk", "sliding") or (window_kind != "full" and window_size < 1):
            raise ValueError(f"Kv8Plan: window '{window_kind}' of {window_size}")
        if len(set(slots)) != len(slots):
            raise ValueError("Kv8Plan: a slot is named twice")
        n = len(starts)
        self.n_seqs, self.n_tokens = n, int(sum(n_new))
        self.window = (window_kind, int(window_size) if window_kind != "full" else 0, int(keep_first) if window_kind == "sliding" else 0)
        ends = [s + m for s, m in zip(starts, n_new)]
        self.width = max(-(-e // BLOCK) for e in ends)
        tables = np.full((2, n, self.width), -1, dtype=np.int32)        # [earlier, exact]
        self.n_earlier = self.most_tiles = 0       # most_tiles: pairs of blocks that a query tile of some sequence meets, at most
        for i, (s, m) in enumerate(zip(starts, n_new)):
            blocks = needed_blocks(s, m, *self.window)
            tables[0, i, blocks] = np.arange(self.n_earlier, self.n_earlier + len(blocks))
            self.n_earlier += len(blocks)
            seen = len(blocks)
            if window_kind != "full":              # a query tile's rows reach back by the window, and to the kept positions
                seen = min(seen, -(-(window_size + 256 + self.window[2]) // BLOCK) + 2)
            self.most_tiles = max(self.most_tiles, seen // 2 + 2)
        at = self.n_earlier
        jobs = []                  # rows of eight numbers: slot, block, first new row, rows, earlier page, exact page, last page, last rows
        for i, (s, e) in enumerate(zip(starts, ends)):
            first, n_blocks = s // BLOCK, -(-e // BLOCK)
            own = np.arange(first, n_blocks)
            tables[1, i, first:n_blocks] = at + own - first
            job = np.empty((len(own), 8), dtype=np.int32)
            job[:, 0], job[:, 1], job[:, 2], job[:, 3] = slots[i], own, 0, np.minimum(BLOCK, e - own * BLOCK)
            job[:, 4], job[:, 5], job[:, 6], job[:, 7] = tables[0, i, first:n_blocks], at + own - first, -1, e - (n_blocks - 1) * BLOCK
            job[0, 2], job[0, 6] = s - first * BLOCK, at + n_blocks - 1 - first       # the first one reads the tail, then keeps it
            jobs.append(job)
            at += n_blocks - first
        for i, s in enumerate(starts):
            earlier = np.flatnonzero(tables[0, i, :s // BLOCK] >= 0)
            job = np.zeros((len(earlier), 8), dtype=np.int32)
            job[:, 0], job[:, 1], job[:, 3], job[:, 4], job[:, 5:7] = slots[i], earlier, BLOCK, tables[0, i, earlier], -1
            jobs.append(job)
        jobs = np.concatenate(jobs)
        self.n_pages, self.n_jobs = at, len(jobs)
        moved = [slot for s, e, slot in zip(starts, ends, slots) if s % BLOCK and e % BLOCK and s // BLOCK != e // BLOCK]
        flat = np.concatenate([tables.ravel(), np.arange(n, dtype=np.int32), jobs.ravel(), np.array(moved, dtype=np.int32)])
        host = torch.from_numpy(flat)
        dev = torch.device(device)
        if dev.type == "cuda":
            host = host.pin_memory()           # (kept below: the copy reads it until it has run)
        self._host, words = host, n * self.width
        d = host.to(dev, non_blocking=True)
        self.earlier_table, self.exact_table = d[:words].view(n, -1), d[words:2 * words].view(n, -1)
        self.seq_ids, self.jobs = d[2 * words:2 * words + n], d[2 * words + n:2 * words + n + jobs.size]
        self.moved = d[2 * words + n + jobs.size:] if moved else None


class KeptTails:
    """Tails that a step gives to other blocks, kept until it is through: a step that fails on the way is undone."""

    def __init__(self):
        self._kept = []

    def keep(self, cache: Kv8Cache, plan: Kv8Plan) -> None:
        """Called before the step's first `kv8_stage`, for the cache of a layer or of many (tensors with one more axis in front)."""
        if plan.moved is not None:
            self._kept += [(t, plan.moved, t.index_select(t.dim() - 4, plan.moved)) for t in (cache.k_tail, cache.v_tail)]

    def put_back(self) -> None:
        for tails, slots, rows in self._kept:
            tails.index_copy_(tails.dim() - 4, slots.long(), rows)
        self._kept.clear()
