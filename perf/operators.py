"""Three operators of serving a decoder, in their plain form (elementary torch operations in 32 bits) and as this library's calls:

  decode     attention of one new token per sequence over a cache held in 8 bits
  prompt     attention of several tokens per sequence over that cache, with the quantisation of the blocks they complete
  logprobs   log probabilities of given tokens, the entropy of each distribution and its most probable tokens

The 8-bit cache.  Positions 64 b .. 64 b + 63 of a sequence are its block b, one page of the cache.  A complete block is held as
8-bit codes with one power of two as scale per page and key/value head, keys and values each; the block of the newest position is held
in bfloat16, in the sequence's tail, until it is complete.  A query sees the keys and values of its own block in bfloat16 and those
of earlier blocks as code times scale.

A case is a dict of plain values.  Attention cases: `kind`, `fmt` ("int8" or "e4m3"), `heads`, `kv_heads`, `dim`, `seqs`, `past`
(positions that the longest sequence has before the step), `ragged` (the sequences' pasts are spread between 0 and `past`, else all are `past`),
`new` (tokens that the longest sequence brings), `window` ("full", "chunk" or "sliding"), `size`, `keep` (first positions that stay visible),
`sink`, `softcap`.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
BLOCK = 64


# ---- the cases -----------------------------------------------------------------------------------------------------
def _attention(name, kind, fmt, heads, kv_heads, dim, seqs, past, *, new=1, ragged=False, window="full", size=0, keep=0, sink=False,
               softcap=0.0):
    return {"name": name, "kind": kind, "fmt": fmt, "heads": heads, "kv_heads": kv_heads, "dim": dim, "seqs": seqs, "past": past, "new": new,
            "ragged": ragged, "window": window, "size": size, "keep": keep, "sink": sink, "softcap": softcap}


def listed():
    return [
        # One short conversation with a small dense decoder: a few pages, latency is all.
        _attention("decode_short", "decode", "int8", 16, 4, 128, 1, 300),
        # The headline benchmark's attention layer, eight sequences whose newest token completes a block.
        _attention("decode_b8_4096", "decode", "int8", 40, 8, 128, 8, 4095),
        # A full server: 64 sequences of unequal lengths up to 16,384 positions, the other format.
        _attention("decode_b64_16k", "decode", "e4m3", 40, 8, 128, 64, 16383, ragged=True),
        # One very long document being asked about.
        _attention("decode_b1_131k", "decode", "int8", 40, 8, 128, 1, 131000),
        # Windowed layers with kept first positions and a sink, small heads, odd lengths.
        _attention("decode_window", "decode", "e4m3", 16, 8, 64, 5, 6001, ragged=True, window="sliding", size=1000, keep=5, sink=True),
        # A short question: a few dozen tokens.
        _attention("prompt_short", "prompt", "int8", 16, 4, 128, 1, 0, new=37),
        # A prompt of an odd length through the headline benchmark's layer.
        _attention("prompt_3001", "prompt", "int8", 40, 8, 128, 1, 0, new=3001),
        # The next turn of a long conversation: a piece of a prompt that starts inside a block.
        _attention("prompt_later", "prompt", "e4m3", 16, 4, 128, 1, 9001, new=509),
        # Four unequal prompts in one step, small heads, windows and soft-capped scores.
        _attention("prompt_window", "prompt", "int8", 16, 8, 64, 4, 700, new=700, ragged=True, window="sliding", size=256, softcap=30.0),
        # The log probability of one token just drawn, with five alternatives.
        {"name": "logprobs_one", "kind": "logprobs", "rows": 1, "vocab": 32000, "top": 5, "dtype": "f32", "masked": False},
        # A decode step's rows at the headline benchmark's vocabulary, with as many alternatives as are commonly asked for.
        {"name": "logprobs_b8", "kind": "logprobs", "rows": 8, "vocab": 202048, "top": 20, "dtype": "f32", "masked": False},
        # Scoring a text: every position of a prompt, no alternatives masked, an odd vocabulary in bfloat16.
        {"name": "logprobs_score", "kind": "logprobs", "rows": 1000, "vocab": 151643, "top": 1, "dtype": "bf16", "masked": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("decode", "decode", "prompt", "logprobs"))
    if kind == "logprobs":
        vocab = _log(rng, 500, 202048)
        return {"kind": kind, "rows": _log(rng, 1, min(2000, 150_000_000 // vocab)), "vocab": vocab, "top": rng.choice((0, 1, 5, 20, 32)),
                "dtype": rng.choice(("f32", "f32", "bf16")), "masked": rng.random() < 0.3}
    kv, dim = rng.choice((1, 2, 4, 8)), rng.choice((64, 128))
    heads = kv * rng.choice((1, 2, 4, 5, 8, 16))
    window = rng.choice(("full", "full", "full", "sliding", "chunk"))
    size = 0 if window == "full" else _log(rng, 30, 3000)
    keep = rng.choice((0, 4, 100)) if window == "sliding" else 0
    more = {"fmt": rng.choice(("int8", "e4m3")), "heads": heads, "kv_heads": kv, "dim": dim, "window": window, "size": size, "keep": keep,
            "sink": rng.random() < 0.3, "softcap": rng.choice((0.0, 0.0, 0.0, 20.0))}
    if kind == "decode":
        seqs = _log(rng, 1, 64)
        return {"kind": kind, **more, "seqs": seqs, "past": _log(rng, 1, min(131000, 500_000 // seqs)), "new": 1, "ragged": rng.random() < 0.6}
    seqs = rng.choice((1, 1, 2, 4))
    new = _log(rng, 2, min(3001, 40000 // heads) // seqs)
    past = rng.choice((0, _log(rng, 1, min(9001, 60_000_000 // (heads * seqs * new)))))
    return {"kind": kind, **more, "seqs": seqs, "past": past, "new": new, "ragged": seqs > 1}


# ---- lengths, the same for everybody -------------------------------------------------------------------------------
def _lengths(case):
    """(positions before the step, tokens that the step brings) per sequence."""
    n = case["seqs"]
    if not case["ragged"] or n == 1:
        return [case["past"]] * n, [case["new"]] * n
    starts = [case["past"] * (i + 1) // n for i in range(n)]
    return starts, [max(1, case["new"] * (n - i) // n) for i in range(n)]


def _visible(case):
    """Pairs of a query and a position that it sees, and the positions of complete blocks and of tails that somebody sees."""
    pairs, old, tail = 0, 0, 0
    for start, new in zip(*_lengths(case)):
        seen_old, seen_tail = 0, 0
        for p in range(start, start + new):
            if case["window"] == "chunk":
                low = p // case["size"] * case["size"]
            else:
                low = max(0, p - case["size"] + 1) if case["window"] == "sliding" else 0
            kept = min(case["keep"], low)
            pairs += p + 1 - low + kept
            if p == start:               # the first query sees what was there, from its window's low end on
                edge = start // BLOCK * BLOCK
                seen_tail = max(0, start - max(low, edge)) + max(0, kept - edge)
                seen_old = max(0, edge - low) + min(kept, edge)
        old, tail = old + seen_old, tail + seen_tail
    return pairs, old, tail


def work(case):
    if case["kind"] == "logprobs":
        n, width = case["rows"] * case["vocab"], 4 if case["dtype"] == "f32" else 2
        return {"bytes": n * width + case["rows"] * (12 + 8 * case["top"]), "flops": 4 * n}
    starts, news = _lengths(case)
    pairs, old, tail = _visible(case)
    tokens, row = sum(news), 2 * case["kv_heads"] * case["dim"]           # elements of a position's key and value rows
    done = sum((s + n) // BLOCK - s // BLOCK for s, n in zip(starts, news)) * BLOCK
    moved = tokens * case["heads"] * case["dim"] * 4 + old * row + tail * row * 2 + tokens * row * 2 + done * row
    return {"bytes": moved, "flops": 4 * pairs * case["heads"] * case["dim"]}


# ---- quantisation, plain -------------------------------------------------------------------------------------------
def _code_type(fmt):
    return torch.int8 if fmt == "int8" else torch.float8_e4m3fn


def _quantise(x, fmt):
    """Codes and scales of blocks x [..., 64, dim]: one power of two for the last two axes."""
    x = x.float()
    top = x.abs().amax((-1, -2))
    exponent = torch.frexp(top).exponent                       # top < 2^exponent, top >= 2^(exponent - 1)
    if fmt == "int8":                                          # the smallest power of two s with top <= 127 s
        exponent = exponent - 7
        exponent = exponent + (top > 127.0 * torch.exp2(exponent.float())).int()
    else:                                                      # top / s in [128, 256)
        exponent = exponent - 8
    exponent = torch.where(top == 0, torch.full_like(exponent, -60), exponent.clamp(-60, 60))
    scale = torch.ldexp(torch.ones_like(top), exponent)
    y = x / scale[..., None, None]
    if fmt == "int8":
        return y.round().clamp(-127, 127).to(torch.int8), scale
    return y.clamp(-448, 448).to(torch.float8_e4m3fn), scale


# ---- inputs --------------------------------------------------------------------------------------------------------
def _rows(g, *shape):
    """Keys, values or queries as layers make them: a few features much larger than the others."""
    x = torch.randn(*shape, generator=g, device=DEV)
    gain = 1.0 + 4.0 * (torch.rand(shape[-1], generator=g, device=DEV) < 0.03).float()
    return (x * gain).to(torch.bfloat16)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    if case["kind"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        x = torch.randn(rows, vocab, generator=g, device=DEV) * 3.0
        if case["masked"]:                                     # tokens that a grammar or a ban rules out
            x.masked_fill_(torch.rand(rows, vocab, generator=g, device=DEV) < 0.1, -math.inf)
        x = x.to(torch.float32 if case["dtype"] == "f32" else torch.bfloat16)
        targets = torch.randint(0, vocab, (rows,), generator=g, device=DEV, dtype=torch.int32)
        return {"case": case, "logits": x, "targets": targets}
    nh, nkv, d, fmt = case["heads"], case["kv_heads"], case["dim"], case["fmt"]
    starts, news = _lengths(case)
    n = len(starts)
    blocks = [-(-(s + m) // BLOCK) for s, m in zip(starts, news)]
    width, tokens = max(blocks), sum(news)
    # every sequence's pages, in a shuffled order of the pool
    order = torch.randperm(sum(blocks), generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(n, width, dtype=torch.int32, device=DEV)
    at = 0
    for i, b in enumerate(blocks):
        table[i, :b] = order[at:at + b]
        at += b
    # the blocks that are complete before the step hold codes; the others are zero until the step completes them
    state = {"case": case, "table": table}
    for name in ("k", "v"):
        codes = torch.zeros(sum(blocks), nkv, BLOCK, d, dtype=_code_type(fmt), device=DEV)
        scales = torch.ones(sum(blocks), nkv, device=DEV)
        for i, s in enumerate(starts):
            for b in range(0, s // BLOCK, 256):
                pages = table[i, b:min(b + 256, s // BLOCK)].long()
                c, sc = _quantise(_rows(g, len(pages), nkv, BLOCK, d), fmt)
                codes.view(torch.uint8)[pages] = c.view(torch.uint8)
                scales[pages] = sc
        state[name], state[name + "_scale"] = codes, scales
        # the newest block so far in bfloat16: rows behind the last position hold whatever an earlier sequence left
        state[name + "_tail"] = _rows(g, n, nkv, BLOCK, d)
    pos = torch.cat([torch.arange(s, s + m, dtype=torch.int32) for s, m in zip(starts, news)]).to(DEV)
    seq = torch.repeat_interleave(torch.arange(n, dtype=torch.int32), torch.tensor(news)).to(DEV)
    state |= {"q": _rows(g, tokens, nh * d), "pos": pos, "seq": seq, "slot": torch.arange(n, dtype=torch.int32, device=DEV),
              "sink": torch.randn(nh, generator=g, device=DEV) if case["sink"] else None, "starts": starts, "news": news,
              "scale": 1.0 / math.sqrt(d), "out": torch.empty(tokens, nh * d, dtype=torch.bfloat16, device=DEV)}
    if case["kind"] == "decode":           # the projection has stored the new token's key and value in the tail
        state["done"] = any(s % BLOCK == BLOCK - 1 for s in starts)
        return state
    # a prompt: the projection has stored the tokens' keys and values in pages of the step's own, from each sequence's
    # first new block on; `exact` names them per sequence and block
    first = [s // BLOCK for s in starts]
    exact = torch.full((n, width), -1, dtype=torch.int32)
    count = 0
    for i in range(n):
        exact[i, first[i]:blocks[i]] = torch.arange(count, count + blocks[i] - first[i])
        count += blocks[i] - first[i]
    state["exact"], state["exact_pages"] = exact.to(DEV), count
    state["new_k"], state["new_v"] = _rows(g, tokens, nkv, d), _rows(g, tokens, nkv, d)
    state["k_tail0"], state["v_tail0"] = state["k_tail"].clone(), state["v_tail"].clone()
    tiles, base = [], 0
    for s, m in zip(starts, news):
        tiles += [(-(s + o + min(256, m - o)), base + o, min(256, m - o)) for o in range(0, m, 256)]
        base += m
    tiles.sort()
    state["tile_tok0"] = torch.tensor([t[1] for t in tiles], dtype=torch.int32, device=DEV)
    state["tile_rows"] = torch.tensor([t[2] for t in tiles], dtype=torch.int32, device=DEV)
    state["first"] = torch.tensor(first, device=DEV)
    if own:
        from cpi_b200.cache.kv8 import Kv8Plan
        plan = Kv8Plan(starts, news, list(range(n)), window_kind=case["window"], window_size=case["size"], keep_first=case["keep"],
                       device=DEV)
        state["plan"] = plan
        for name in ("k", "v"):
            pages = torch.zeros(plan.n_pages, nkv, BLOCK, d, dtype=torch.bfloat16, device=DEV)
            pages[plan.n_earlier + exact.to(DEV)[seq.long(), (pos // BLOCK).long()].long(), :, (pos % BLOCK).long()] = state["new_" + name]
            state[name + "_pages"] = pages
    return state


# ---- plain forms ---------------------------------------------------------------------------------------------------
def _low(case, pos):
    if case["window"] == "chunk":
        return pos // case["size"] * case["size"]
    return (pos - case["size"] + 1).clamp_min(0) if case["window"] == "sliding" else torch.zeros_like(pos)


def _softmax_values(s, case, state, keys_seen, values):
    """Scores s [b, kv heads, group, queries, keys] -> outputs, all in 32 bits; a sink joins the sums."""
    s = s * state["scale"]
    if case["softcap"]:
        s = case["softcap"] * torch.tanh(s / case["softcap"])
    s = s.masked_fill(~keys_seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    if state["sink"] is not None:
        sink = state["sink"].view(1, case["kv_heads"], -1, 1, 1)
        top = torch.maximum(top, sink)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    if state["sink"] is not None:
        total = total + torch.exp(sink - top)
    return torch.matmul(p, values[:, :, None]) / total


def _dequantised(state, name, table):
    """[sequences, kv heads, blocks * 64, dim] in 32 bits: code times scale."""
    pages = table.clamp_min(0).long()
    x = state[name][pages].float() * state[name + "_scale"][pages][..., None, None]
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)


def _decode_plain(state):
    case = state["case"]
    nkv, d = case["kv_heads"], case["dim"]
    pos, table = state["pos"], state["table"]
    n, width = table.shape
    q = state["q"].float().view(n, nkv, -1, 1, d)
    at = torch.arange(width * BLOCK, device=DEV)[None]
    edge, low = pos // BLOCK * BLOCK, _low(case, pos)
    see = lambda j: ((j >= low[:, None]) | (j < case["keep"])) & (j <= pos[:, None])          # noqa: E731
    own_at = edge[:, None] + torch.arange(BLOCK, device=DEV)[None]
    k = torch.cat([_dequantised(state, "k", table), state["k_tail"].float()], 2)
    s = torch.matmul(q, k[:, :, None].transpose(-1, -2))
    k = None
    seen = torch.cat([see(at) & (at < edge[:, None]), see(own_at)], 1)[:, None]
    v = torch.cat([_dequantised(state, "v", table), state["v_tail"].float()], 2)
    v = v.masked_fill(~seen[:, 0, :, None][:, None], 0.0)
    out = _softmax_values(s, case, state, seen, v)
    result = {"out": out.reshape(n, -1).to(torch.bfloat16)}
    if state["done"]:                      # tokens that complete a block: its codes and scales go to the cache
        full = pos % BLOCK == BLOCK - 1
        pages = table[full.nonzero().flatten(), (pos[full] // BLOCK).long()].long()
        for name in ("k", "v"):
            c, sc = _quantise(state[name + "_tail"][full], case["fmt"])
            codes, scales = state[name].clone(), state[name + "_scale"].clone()
            codes.view(torch.uint8)[pages] = c.view(torch.uint8)
            scales[pages] = sc
            result[name], result[name + "_scale"] = codes, scales
    return result


def _prompt_plain(state):
    case = state["case"]
    nkv, d, fmt = case["kv_heads"], case["dim"], case["fmt"]
    table, exact, pos, seq = state["table"], state["exact"], state["pos"], state["seq"].long()
    n, width = table.shape
    starts, news = torch.tensor(state["starts"], device=DEV), torch.tensor(state["news"], device=DEV)
    end = starts + news
    result = {}
    held = {}
    for name in ("k", "v"):
        # the step's own blocks in bfloat16: the tail's rows, then the new ones
        pages = torch.zeros(state["exact_pages"], nkv, BLOCK, d, dtype=torch.bfloat16, device=DEV)
        begun = starts % BLOCK > 0
        rows = torch.arange(BLOCK, device=DEV)[None] < (starts % BLOCK)[:, None]
        first_page = exact[torch.arange(n, device=DEV), state["first"]].long()
        pages[first_page] = torch.where(rows[:, None, :, None], state[name + "_tail0"], torch.zeros((), dtype=torch.bfloat16, device=DEV))
        pages[exact[seq, (pos // BLOCK).long()].long(), :, (pos % BLOCK).long()] = state["new_" + name]
        # complete blocks go to the cache
        block_end = (torch.arange(width, device=DEV)[None] + 1) * BLOCK
        whole = (exact >= 0) & (block_end <= end[:, None])
        codes, scales = state[name].clone(), state[name + "_scale"].clone()
        c, sc = _quantise(pages[exact[whole].long()], fmt)
        codes.view(torch.uint8)[table[whole].long()] = c.view(torch.uint8)
        scales[table[whole].long()] = sc
        result[name], result[name + "_scale"] = codes, scales
        # a sequence whose last block is not complete keeps its rows in the tail
        last = ((end - 1) // BLOCK).clamp_min(0)
        open_rows = (torch.arange(BLOCK, device=DEV)[None] < (end % BLOCK)[:, None])[:, None, :, None]
        last_page = exact[torch.arange(n, device=DEV), last].long()
        result[name + "_tail"] = torch.where(open_rows, pages[last_page], state[name + "_tail0"])
        x = pages[exact.clamp_min(0).long()].float().masked_fill((exact < 0)[:, :, None, None, None], 0.0)
        held[name + "_exact"] = x.permute(0, 2, 1, 3, 4).flatten(2, 3)
        held[name + "_earlier"] = _dequantised({name: codes, name + "_scale": scales}, name, table)
    # queries padded to the longest sequence
    most = max(state["news"])
    offset = pos - starts[seq].int()
    q = torch.zeros(n, most, case["heads"] * d, device=DEV)
    q[seq, offset.long()] = state["q"].float()
    q = q.view(n, most, nkv, -1, d).permute(0, 2, 3, 1, 4)
    qpos = starts[:, None] + torch.arange(most, device=DEV)[None]
    at = torch.arange(width * BLOCK, device=DEV)[None, None]
    low, edge = _low(case, qpos)[..., None], (qpos // BLOCK * BLOCK)[..., None]
    see = ((at >= low) | (at < case["keep"])) & (at <= qpos[..., None])
    seen = torch.cat([see & (at < edge), see & (at >= edge)], -1)
    s = torch.matmul(q, torch.cat([held["k_earlier"], held["k_exact"]], 2)[:, :, None].transpose(-1, -2))
    out = _softmax_values(s, case, state, seen, torch.cat([held["v_earlier"], held["v_exact"]], 2))
    out = out.permute(0, 3, 1, 2, 4).reshape(n, most, -1)[seq, offset.long()]
    return {"out": out.to(torch.bfloat16), **result}


def _logprobs_plain(state):
    case = state["case"]
    x = state["logits"].float()
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    lse = top + torch.log(total)
    chosen = x.gather(-1, state["targets"].long()[:, None]) - lse
    spread = torch.where(e > 0, e * (x - top), torch.zeros_like(e)).sum(-1) / total[:, 0]
    result = {"logprob": chosen[:, 0], "entropy": torch.log(total[:, 0]) - spread}
    if case["top"]:
        values, ids = torch.sort(x, dim=-1, descending=True, stable=True)
        result["top_logprobs"] = values[:, :case["top"]] - lse
        result["top_ids"] = ids[:, :case["top"]].int()
    return result


# ---- one pass ------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if not own:
        return {"decode": _decode_plain, "prompt": _prompt_plain, "logprobs": _logprobs_plain}[case["kind"]](state)
    from cpi_b200.csrc import lib as K
    if case["kind"] == "logprobs":
        got = K.log_probs(state["logits"], state["targets"], top=case["top"])
        result = {"logprob": got.logprob, "entropy": got.entropy}
        if case["top"]:
            result |= {"top_logprobs": got.top_logprobs, "top_ids": got.top_ids}
        return result
    from cpi_b200.cache.kv8 import Kv8Cache
    cache = Kv8Cache(state["k"], state["v"], state["k_scale"], state["v_scale"], state["k_tail"], state["v_tail"])
    how = {"n_heads": case["heads"], "scale": state["scale"], "window_kind": K.WINDOW_KINDS[case["window"]], "window_size": case["size"],
           "keep_first": case["keep"], "sink": state["sink"], "softcap": case["softcap"]}
    if case["kind"] == "decode":
        K.attention_decode_kv8(state["q"], state["out"], cache, state["table"], state["seq"], state["pos"], state["slot"],
                               max_context=max(state["starts"]) + 1, **how)
        result = {"out": state["out"]}
        if state["done"]:
            result |= {"k": state["k"], "k_scale": state["k_scale"], "v": state["v"], "v_scale": state["v_scale"]}
        return result
    if any(s % BLOCK for s in state["starts"]):           # (so that a second pass meets the same tails)
        state["k_tail"].copy_(state["k_tail0"])
        state["v_tail"].copy_(state["v_tail0"])
    K.kv8_stage(cache, state["table"], state["plan"], state["k_pages"], state["v_pages"])
    K.attention_prefill_kv8(state["q"], state["out"], state["k_pages"], state["v_pages"], state["plan"], state["seq"], state["pos"],
                            state["tile_tok0"], state["tile_rows"], **how)
    return {"out": state["out"], **{k: state[k] for k in ("k", "k_scale", "k_tail", "v", "v_scale", "v_tail")}}


# ---- from the definitions, in 64 bits, a sequence and a key/value head at a time ------------------------------------
def _held64(x, fmt):
    """The values that blocks x [blocks, 64, dim] stand for once they are held in 8 bits, in 64 bits."""
    x = x.double()
    top = x.abs().flatten(1).amax(1)
    powers = torch.arange(-60, 61, device=DEV, dtype=torch.float64)
    if fmt == "int8":                      # the smallest power of two that covers the block with codes up to 127
        covers = 127.0 * torch.exp2(powers)[None] >= top[:, None]
    else:                                  # the smallest one of which the block's largest value is less than 256 times as much
        covers = 256.0 * torch.exp2(powers)[None] > top[:, None]
    scale = torch.exp2(powers)[covers.int().argmax(1)][:, None, None]
    y = x / scale
    if fmt == "int8":
        return torch.round(y) * scale
    # four significant bits, the last one worth 2^-9 or more
    step = torch.exp2((torch.frexp(y.abs().clamp_min(2.0 ** -30)).exponent - 4).clamp_min(-9).double())
    return torch.round(y / step) * step * scale


def _exact_attention(case, state):
    nkv, d, group = case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"]
    out = torch.empty_like(state["q"], dtype=torch.float64)
    base = 0
    for i, (start, new) in enumerate(zip(state["starts"], state["news"])):
        q = state["q"][base:base + new].double().view(new, nkv, group, d)
        first, n_blocks = start // BLOCK, -(-(start + new) // BLOCK)
        p = torch.arange(start, start + new, device=DEV)[:, None]
        j = torch.arange(n_blocks * BLOCK, device=DEV)[None]
        seen = j <= p
        if case["window"] == "chunk":
            seen &= j // case["size"] == p // case["size"]
        elif case["window"] == "sliding":
            seen &= (p - j < case["size"]) | (j < case["keep"])
        same = j // BLOCK == p // BLOCK
        pages = state["table"][i, :n_blocks].long()
        for h in range(nkv):
            near, far = [], []
            for name in ("k", "v"):
                rows = torch.zeros(n_blocks * BLOCK, d, dtype=torch.bfloat16, device=DEV)
                tail = state[name + "_tail"] if case["kind"] == "decode" else state[name + "_tail0"]
                have = start % BLOCK + (new if case["kind"] == "decode" else 0)
                rows[first * BLOCK:first * BLOCK + have] = tail[i, h, :have]
                if case["kind"] == "prompt":
                    rows[start:start + new] = state["new_" + name][base:base + new, h]
                value = state[name][pages[:first], h].double() * state[name + "_scale"][pages[:first], h].double()[:, None, None]
                later = _held64(rows[first * BLOCK:].view(-1, BLOCK, d), case["fmt"])
                near.append(rows.double())
                far.append(torch.cat([value, later]).view(-1, d))
            s = torch.einsum("tgd,jd->gtj", q[:, h], far[0])
            s = torch.where(same, torch.einsum("tgd,jd->gtj", q[:, h], near[0]), s) * state["scale"]
            if case["softcap"]:
                s = case["softcap"] * torch.tanh(s / case["softcap"])
            s = torch.where(seen, s, torch.full_like(s, -math.inf))
            if state["sink"] is not None:
                s = torch.cat([s, state["sink"][h * group:(h + 1) * group].double()[:, None, None].expand(-1, new, 1)], -1)
            w = torch.softmax(s, -1)[..., :n_blocks * BLOCK]
            o = torch.einsum("gtj,jd->tgd", torch.where(same, torch.zeros_like(w), w), far[1])
            o += torch.einsum("gtj,jd->tgd", torch.where(same, w, torch.zeros_like(w)), near[1])
            out.view(-1, nkv, group, d)[base:base + new, h] = o
        base += new
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] != "logprobs":
        if work(case)["flops"] > 4e11:
            return None
        return {"out": _exact_attention(case, state)}
    parts = {"logprob": [], "entropy": [], "top_logprobs": []}
    for r in range(case["rows"]):
        lp = torch.log_softmax(state["logits"][r].double(), -1)
        p = lp.exp()
        parts["logprob"].append(lp[state["targets"][r].long()])
        parts["entropy"].append(-(p * torch.where(p > 0, lp, torch.zeros_like(lp))).sum())
        parts["top_logprobs"].append(torch.topk(lp, case["top"]).values if case["top"] else lp[:0])
    if not case["top"]:
        del parts["top_logprobs"]
    return {k: torch.stack(v) for k, v in parts.items()}
