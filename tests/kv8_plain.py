"""The cache in 8 bits and the attention over it in plain 64-bit arithmetic, one query at a time, for the tests.

`Sequence` is what a sequence has: every position's key and value in bfloat16.  What a query sees follows from them alone:
its own block of 64 positions as they are, complete earlier blocks as held in 8 bits."""
from __future__ import annotations

import math

import torch

BLOCK = 64
TYPES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def scale_of(top: float, fmt: str) -> float:
    if top == 0.0:
        return 2.0 ** -60
    if fmt == "int8":
        e = -60
        while e < 60 and 127.0 * 2.0 ** e < top:
            e += 1
        return 2.0 ** e
    e = math.floor(math.log2(top))
    assert 2.0 ** e <= top < 2.0 ** (e + 1)
    return 2.0 ** max(-60, min(60, e - 7))


def nearest_e4m3(y: torch.Tensor) -> torch.Tensor:
    """The nearest e4m3 numbers (ties to even) of 64-bit numbers, saturating at 448; NaN stays."""
    y = y.clamp(-1e6, 1e6)              # (an infinity saturates too)
    a = y.abs()
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(a.clamp_min(2.0 ** -40))), min=-6.0) - 3)
    out = torch.round(a / step) * step
    return torch.where(y.isnan(), y, torch.copysign(out.clamp_max(448.0), y))


def hold(block: torch.Tensor, fmt: str):
    """(codes as 64-bit numbers, scale) of one block [64, dim] of one head."""
    x = block.double()
    finite = x[x.isfinite()]
    s = scale_of(float(finite.abs().max()) if finite.numel() else 0.0, fmt)
    y = x / s
    if fmt == "int8":
        c = torch.round(y.nan_to_num(0.0, posinf=1e9, neginf=-1e9)).clamp(-127, 127)
    else:
        c = nearest_e4m3(y)
    return c, s


def low(pos: int, window: str, size: int) -> int:
    return pos // size * size if window == "chunk" else max(0, pos - size + 1) if window == "sliding" else 0


def rows_seen(pos, window, size, keep):
    first = low(pos, window, size)
    kept = min(keep, first) if window == "sliding" else 0
    return list(range(kept)) + list(range(first, pos + 1))


def held_rows(x: torch.Tensor, fmt: str) -> torch.Tensor:
    """What complete blocks of x [positions, heads, dim] stand for (64 bits); rows of an incomplete one stay."""
    out = x.double().clone()
    for b in range(x.shape[0] // BLOCK):
        for h in range(x.shape[1]):
            c, s = hold(x[b * BLOCK:(b + 1) * BLOCK, h], fmt)
            out[b * BLOCK:(b + 1) * BLOCK, h] = c * s
    return out


def attend(q, k, v, positions, *, fmt, scale, window="full", size=0, keep=0, sink=None, softcap=0.0):
    """q [len(positions), heads, dim]; k, v [length, kv heads, dim] bfloat16.  Returns (outputs, sum p |v| / Z), both
    [queries, heads, dim] in 64 bits: the second bounds what rounding the probabilities can do."""
    nh, nkv = q.shape[1], k.shape[1]
    hk, hv = held_rows(k, fmt), held_rows(v, fmt)
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    for i, pos in enumerate(positions):
        if pos < 0:
            continue
        at = torch.tensor(rows_seen(pos, window, size, keep), device=q.device)
        near = (at >= pos // BLOCK * BLOCK)[:, None, None]
        kk = torch.where(near, k[at].double(), hk[at]).repeat_interleave(nh // nkv, 1)
        vv = torch.where(near, v[at].double(), hv[at]).repeat_interleave(nh // nkv, 1)
        s = torch.einsum("hd,jhd->hj", q[i].double(), kk) * scale
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        if sink is not None:
            s = torch.cat([s, sink.double()[:, None]], 1)
        p = torch.softmax(s, 1)[:, :len(at)]
        out[i] = torch.einsum("hj,jhd->hd", p, vv)
        mag[i] = torch.einsum("hj,jhd->hd", p, vv.abs()) + 2.0 ** 8 * floor(p, at, hv, pos // BLOCK * BLOCK, nh // nkv)
    return out, mag


def floor(p, at, held, edge, group):
    """What the float16 probabilities of single tokens may be off by whatever their size, as an output [heads, 1].  A kernel
    multiplies a block's codes c by float16 numbers P = p 2^e x (2^e the block's scale, x the same for all), the largest of which
    is 2^6 or more; float16 numbers are at most 2^-25 from what they round (half the step of its smallest ones), so a term is off
    by 2^-25 |c| beside a largest P of 2^6: by 2^-31 |c| max(p 2^e).  |c| is below 2^9, and max(p 2^e) |c| at most 2^2 times
    max(p m), m the largest held number of p's block, for |c| <= 2^8 m / 2^e / 2^6: int8 codes reach 64 or more, e4m3 codes 128."""
    m = torch.zeros_like(p)
    far = at < edge
    if not far.any():
        return torch.zeros(p.shape[0], 1, dtype=p.dtype, device=p.device)
    blocks = at // BLOCK
    for b in blocks[far].unique().tolist():
        top = held[b * BLOCK:(b + 1) * BLOCK].abs().amax((0, 2)).repeat_interleave(group)          # per head
        m[:, blocks == b] = top[:, None]
    return int(far.sum()) * 2.0 ** -31 * 2.0 ** 2 * (p * m * far).amax(1, keepdim=True)


def tolerance(out, mag):
    """The output is rounded to bfloat16 (2^-8 of its value); probabilities are rounded to bfloat16 or finer before they are
    multiplied (2^-8 of each term's size, so of their sum; `floor` below that); scores, exponentials and sums are float32 (2^-10 of the terms' size
    covers scores up to 1,000)."""
    return 2.0 ** -8 * out.abs() + (2.0 ** -8 + 2.0 ** -10) * mag + 1e-30
