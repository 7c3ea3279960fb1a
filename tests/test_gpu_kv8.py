"""The cache in 8 bits: what is stored, attention of single tokens and of prompts over it, against plain 64-bit arithmetic."""
from __future__ import annotations

import math

import pytest
import torch

import kv8_plain as P
from cpi_b200.cache.kv8 import FORMATS, Kv8Cache, Kv8Plan
from cpi_b200.csrc import lib as K
from cpi_b200.engine.batch import BatchStager

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BLOCK = 64


class Rig:
    """A cache and sequences whose every key and value is known; steps go through the kernels."""

    def __init__(self, lengths, *, fmt="int8", nh=8, nkv=2, d=128, seed=0, slots=None, spare=3, garbage=True, gain=1.0):
        self.g = torch.Generator(device=DEV).manual_seed(seed)
        self.fmt, self.nh, self.nkv, self.d = fmt, nh, nkv, d
        n = len(lengths)
        self.slots = list(slots) if slots is not None else list(reversed(range(n)))
        n_slots = max(self.slots) + 1 + spare
        width = max(-(-length // BLOCK) for length in lengths) + 1
        n_pages = n * width + spare
        perm = torch.randperm(n_pages, generator=self.g, device=DEV)[:n * width].int().view(n, width)
        self.table = torch.zeros(n_slots, width, dtype=torch.int32, device=DEV)
        for i, s in enumerate(self.slots):
            self.table[s] = perm[i]
        shape = (n_pages, nkv, BLOCK, d)
        kind = FORMATS[fmt]
        # what earlier sequences left: codes of any value (e4m3 NaN among them), scales, tails with NaN and infinities
        code = lambda: torch.randint(0, 256, shape, generator=self.g, device=DEV, dtype=torch.uint8).view(kind)       # noqa: E731
        tail = lambda: torch.full((n_slots, nkv, BLOCK, d), math.nan if garbage else 0.0, device=DEV).bfloat16()       # noqa: E731
        self.cache = Kv8Cache(code(), code(), torch.full((n_pages, nkv), 2.0, device=DEV), torch.full((n_pages, nkv), 0.5, device=DEV),
                              tail(), tail())
        self.k = [self.rows(length, nkv, d) * gain for length in lengths]
        self.v = [self.rows(length, nkv, d) * gain for length in lengths]
        self.done = [0] * n
        self.stager = BatchStager(torch.device(DEV))

    def rows(self, *shape):
        x = torch.randn(*shape, generator=self.g, device=DEV)
        x = x * (1.0 + 6.0 * (torch.rand(shape[-1], generator=self.g, device=DEV) < 0.05).float())
        return x.bfloat16()

    def load(self, i, length):
        """Puts the first `length` positions of sequence i into the cache with plain torch."""
        for b in range(length // BLOCK):
            page = int(self.table[self.slots[i], b])
            for h in range(self.nkv):
                for x, codes, scales in ((self.k[i], self.cache.k, self.cache.k_scale), (self.v[i], self.cache.v, self.cache.v_scale)):
                    c, s = P.hold(x[b * BLOCK:(b + 1) * BLOCK, h], self.fmt)
                    codes.view(torch.uint8)[page, h] = c.to(FORMATS[self.fmt]).view(torch.uint8)
                    scales[page, h] = s
        r = length % BLOCK
        if r:
            self.cache.k_tail[self.slots[i], :, :r] = self.k[i][length - r:length].transpose(0, 1)
            self.cache.v_tail[self.slots[i], :, :r] = self.v[i][length - r:length].transpose(0, 1)
        self.done[i] = length

    def store_newest(self, i, pos):
        self.cache.k_tail[self.slots[i], :, pos % BLOCK] = self.k[i][pos]
        self.cache.v_tail[self.slots[i], :, pos % BLOCK] = self.v[i][pos]

    def decode(self, positions, *, window="full", size=0, keep=0, sink=None, softcap=0.0, q=None, max_context=None, stored=True):
        if stored:
            for i, pos in enumerate(positions):
                if pos >= 0:
                    self.store_newest(i, pos)
        n = len(positions)
        q = self.rows(n, self.nh, self.d) if q is None else q
        out = torch.full((n, self.nh * self.d), 7.0, dtype=torch.bfloat16, device=DEV)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)       # noqa: E731
        K.attention_decode_kv8(q.view(n, -1), out, self.cache, self.table, i32(list(range(n))), i32(positions), i32(self.slots),
                               n_heads=self.nh, scale=self.d ** -0.5, max_context=max_context or max(max(positions) + 1, 1),
                               window_kind=K.WINDOW_KINDS[window], window_size=size, keep_first=keep, sink=sink, softcap=softcap)
        torch.cuda.synchronize()
        return q, out.view(n, self.nh, self.d)

    def prompt(self, news, *, window="full", size=0, keep=0, sink=None, softcap=0.0, plan=None):
        """Every sequence i brings news[i] tokens; returns queries and outputs per sequence."""
        starts = list(self.done)
        n, T = len(news), sum(news)
        batch = self.stager.stage(self.slots, starts, [[0] * m for m in news], [[]] * n, torch.bfloat16)
        plan = plan or Kv8Plan(starts, news, self.slots, window_kind=window, window_size=size, keep_first=keep, device=DEV)
        kp = torch.full((plan.n_pages, self.nkv, BLOCK, self.d), math.nan, device=DEV).bfloat16()
        vp = kp.clone()
        at = plan.exact_table.long()[batch.token_seq.long(), (batch.token_pos // BLOCK).long()]
        row = (batch.token_pos % BLOCK).long()
        kp[at, :, row] = torch.cat([k[s:s + m] for k, s, m in zip(self.k, starts, news)])
        vp[at, :, row] = torch.cat([v[s:s + m] for v, s, m in zip(self.v, starts, news)])
        q = self.rows(T, self.nh, self.d)
        out = torch.full((T + 1, self.nh * self.d), 7.0, dtype=torch.bfloat16, device=DEV)
        K.kv8_stage(self.cache, self.table, plan, kp, vp)
        K.attention_prefill_kv8(q.view(T, -1), out[:T], kp, vp, plan, batch.token_seq, batch.token_pos, batch.tile_tok0, batch.tile_rows,
                                n_heads=self.nh, scale=self.d ** -0.5, window_kind=K.WINDOW_KINDS[window], window_size=size, keep_first=keep,
                                sink=sink, softcap=softcap)
        torch.cuda.synchronize()
        assert (out[T] == 7.0).all(), "rows behind the last token were written"
        self.done = [s + m for s, m in zip(starts, news)]
        return q.split(list(news)), out[:T].view(T, self.nh, self.d).split(list(news)), starts

    def check(self, i, q, out, positions, **how):
        ref, mag = P.attend(q, self.k[i], self.v[i], positions, fmt=self.fmt, scale=self.d ** -0.5, **how)
        err = (out.double() - ref).abs()
        assert not out.isnan().any()
        bad = err > P.tolerance(ref, mag)
        assert not bad.any(), f"sequence {i}: off by {float(err[bad].max()):.3e} at {bad.nonzero()[0].tolist()}"

    def check_held(self, i):
        """The cache holds what the first done[i] positions are held as, bit for bit, and the tail the open block's rows."""
        n = self.done[i]
        for b in range(n // BLOCK):
            page = int(self.table[self.slots[i], b])
            for h in range(self.nkv):
                for x, codes, scales in ((self.k[i], self.cache.k, self.cache.k_scale), (self.v[i], self.cache.v, self.cache.v_scale)):
                    c, s = P.hold(x[b * BLOCK:(b + 1) * BLOCK, h], self.fmt)
                    assert float(scales[page, h]) == s
                    got = codes[page, h].float().double()
                    assert torch.equal(got.nan_to_num(1e9), c.nan_to_num(1e9)), f"block {b} head {h}"
        r = n % BLOCK
        if r:
            assert torch.equal(self.cache.k_tail[self.slots[i], :, :r], self.k[i][n - r:n].transpose(0, 1))
            assert torch.equal(self.cache.v_tail[self.slots[i], :, :r], self.v[i][n - r:n].transpose(0, 1))


WINDOWS = [dict(), dict(window="sliding", size=100), dict(window="sliding", size=70, keep=5), dict(window="sliding", size=1),
           dict(window="sliding", size=130, keep=200), dict(window="chunk", size=96), dict(window="chunk", size=64)]


# ---- single tokens -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("nh,nkv,d", [(8, 2, 128), (5, 1, 64), (16, 1, 128), (12, 1, 64), (3, 3, 128), (40, 8, 128)])
def test_single_tokens(fmt, nh, nkv, d):
    positions = [0, 1, 15, 16, 62, 63, 64, 65, 127, 128, 200, 511, 700]
    rig = Rig([p + 1 for p in positions], fmt=fmt, nh=nh, nkv=nkv, d=d, seed=d + nh)
    for i, p in enumerate(positions):
        rig.load(i, p)
    q, out = rig.decode(positions)
    for i, p in enumerate(positions):
        rig.check(i, q[i:i + 1], out[i:i + 1], [p])
        rig.done[i] = p + 1
        rig.check_held(i)          # 63, 127, 511 complete a block


@pytest.mark.parametrize("how", WINDOWS)
@pytest.mark.parametrize("fmt,nh,nkv,d", [("int8", 8, 2, 128), ("e4m3", 12, 1, 64)])
def test_single_tokens_windows(how, fmt, nh, nkv, d):
    positions = [0, 40, 63, 64, 95, 96, 130, 255, 300, 449]
    rig = Rig([p + 1 for p in positions], fmt=fmt, nh=nh, nkv=nkv, d=d, seed=3)
    for i, p in enumerate(positions):
        rig.load(i, p)
    q, out = rig.decode(positions, **how)
    for i, p in enumerate(positions):
        rig.check(i, q[i:i + 1], out[i:i + 1], [p], **how)


@pytest.mark.parametrize("sink", [False, True])
@pytest.mark.parametrize("softcap", [0.0, 5.0])
@pytest.mark.parametrize("max_context", [1, 100000])
def test_single_tokens_sink_and_cap(sink, softcap, max_context):
    """`max_context` only divides the work: one block of threads, or more of them than there are pages."""
    positions = [0, 63, 500, 1200]
    rig = Rig([p + 1 for p in positions], nh=8, nkv=2, seed=4)
    rig.table = torch.nn.functional.pad(rig.table, (0, 2000))
    sink = torch.tensor([-3.0, 0.0, 5.0, 200.0, -200.0, 1.0, 2.0, 3.0], device=DEV) if sink else None
    for i, p in enumerate(positions):
        rig.load(i, p)
    q, out = rig.decode(positions, sink=sink, softcap=softcap, max_context=max_context)
    for i, p in enumerate(positions):
        rig.check(i, q[i:i + 1], out[i:i + 1], [p], sink=sink, softcap=softcap)


@pytest.mark.parametrize("nh,d,splits", [(4, 64, s) for s in range(1, 10)] + [(5, 128, 3), (16, 128, 2), (12, 64, 7), (16, 128, 8), (8, 128, 17), (9, 128, 20),
                                         (4, 64, 35)])
def test_splits_of_the_keys(nh, d, splits):
    """One block of threads, clusters of any size, and blocks that a second kernel joins, with few heads and with two tiles of them."""
    p = (4 * splits - 1) * 64 - 7
    assert K._kv8_splits(0, 1, -(-(p + 1) // 64))[0] == splits
    rig = Rig([p + 1], fmt="e4m3", nh=nh, nkv=1, d=d, seed=5)
    rig.load(0, p)
    sink = torch.linspace(-3, 9, nh, device=DEV) if splits % 2 else None
    q, out = rig.decode([p], sink=sink)
    rig.check(0, q, out, [p], sink=sink)


def test_scales_that_are_no_powers_of_two():
    """Codes of another maker: any positive scales."""
    p = 200
    rig = Rig([p + 1], nh=4, nkv=2, d=64, seed=31)
    rig.load(0, p)
    rig.cache.k_scale.mul_(1.37)
    rig.cache.v_scale.mul_(0.71)
    q, out = rig.decode([p])
    held = {}
    for name in ("k", "v"):
        x = getattr(rig, name)[0].double()
        for b in range(3):
            page = int(rig.table[rig.slots[0], b])
            codes, scales = getattr(rig.cache, name)[page].double(), getattr(rig.cache, name + "_scale")[page].double()
            x[b * 64:(b + 1) * 64] = (codes * scales[:, None, None]).transpose(0, 1)
        held[name] = x.repeat_interleave(2, 1)
    s = torch.softmax(torch.einsum("hd,jhd->hj", q[0].double(), held["k"]) / 8.0, 1)
    ref, mag = torch.einsum("hj,jhd->hd", s, held["v"]), torch.einsum("hj,jhd->hd", s, held["v"].abs())
    assert ((out[0].double() - ref).abs() <= P.tolerance(ref, mag)).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("gain", [1e-12, 1e-3, 30.0, 1e6])
def test_scales_far_apart(fmt, gain):
    """Blocks whose values differ by many powers of two share an accumulator; queries of any size."""
    p = 320
    rig = Rig([p + 1], fmt=fmt, nh=8, nkv=2, seed=6)
    for b in range(5):
        rig.v[0][b * 64:(b + 1) * 64] *= gain ** (b % 3 - 1)
    rig.v[0][64:128] = 0.0
    rig.load(0, p)
    q, out = rig.decode([p], q=rig.rows(1, 8, 128) * (1.0 if gain > 1 else 3.0))
    rig.check(0, q, out, [p])
    small = rig.rows(1, 8, 128) * 1e-30
    q, out = rig.decode([p], q=small)
    rig.check(0, q, out, [p])


def test_padded_rows_and_wrong_indices():
    """A position below zero: zeros.  Slots, positions and pages outside the cache: zeros where nothing can be read, the
    error flag, and nothing written."""
    rig = Rig([100, 64, 200], seed=7)
    for i, p in enumerate([99, 63, 199]):
        rig.load(i, p)
    before = [t.clone().view(torch.uint8) for t in rig.cache]
    q, out = rig.decode([99, -1, 199])
    assert (out[1] == 0).all()
    rig.check(0, q[:1], out[:1], [99])
    rig.check(2, q[2:], out[2:], [199])
    flags = K.device_error_flags(DEV)
    assert int(flags[0]) == 0
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)       # noqa: E731
    out2 = torch.full((3, 8 * 128), 7.0, dtype=torch.bfloat16, device=DEV)
    K.attention_decode_kv8(q.view(3, -1), out2, rig.cache, rig.table, i32([0, 5, 2]), i32([100000, 63, 199]), i32([2, 1, 9]), n_heads=8,
                           scale=0.1, max_context=256)
    torch.cuda.synchronize()
    assert (out2 == 0).all() and int(flags[0]) != 0
    flags.zero_()
    for i in (0, 2):
        rig.store_newest(i, [99, 63, 199][i])
    after = [t.clone().view(torch.uint8) for t in rig.cache]
    same = [torch.equal(a, b) for a, b in zip(before[:4], after[:4])]
    assert all(same)
    bad = rig.table.clone()
    bad[rig.slots[2], 1] = 10 ** 6
    K.attention_decode_kv8(q.view(3, -1), out2, rig.cache, bad, i32([0, 1, 2]), i32([99, -1, 199]), i32(rig.slots), n_heads=8, scale=128 ** -0.5,
                           max_context=256)
    torch.cuda.synchronize()
    assert int(flags[0]) != 0
    flags.zero_()
    rig.check(0, q[:1], out2[:1].view(1, 8, 128), [99])


def test_prompt_indices_outside_of_the_step():
    """Tiles, sequences and positions that the plan does not have: the error word, and nothing outside of the output is touched."""
    rig = Rig([300, 200], seed=9)
    flags = K.device_error_flags(DEV)
    assert int(flags[0]) == 0
    starts, news = [0, 0], [300, 200]
    batch = rig.stager.stage(rig.slots, starts, [[0] * m for m in news], [[], []], torch.bfloat16)
    plan = Kv8Plan(starts, news, rig.slots, device=DEV)
    kp = torch.zeros(plan.n_pages, 2, 64, 128, dtype=torch.bfloat16, device=DEV)
    vp, q = kp.clone(), rig.rows(500, 8 * 128)
    store = torch.full((502, 8 * 128), 7.0, dtype=torch.bfloat16, device=DEV)
    out = store[1:501]
    good = dict(token_seq=batch.token_seq, token_pos=batch.token_pos, tile_tok0=batch.tile_tok0, tile_rows=batch.tile_rows)
    for bad in (dict(tile_tok0=batch.tile_tok0 + 400), dict(tile_tok0=batch.tile_tok0 - 300), dict(tile_rows=batch.tile_rows * 1000),
                dict(tile_rows=batch.tile_rows * 0), dict(token_seq=batch.token_seq + 7), dict(token_seq=batch.token_seq - 3),
                dict(token_pos=batch.token_pos + 10 ** 6), dict(token_pos=batch.token_pos - 10 ** 6), dict()):
        K.attention_prefill_kv8(q, out, kp, vp, plan, **{**good, **bad}, n_heads=8, scale=0.1)
        torch.cuda.synchronize()
        assert int(flags[0]) == (3 if bad else 0), bad.keys()
        flags.zero_()
        assert (store[0] == 7.0).all() and (store[501] == 7.0).all()


def test_infinities_and_nan_in_masked_places():
    """What a query does not see may hold anything: rows behind the newest (the Rig's tails), blocks before a window."""
    p = 400
    rig = Rig([p + 1], fmt="e4m3", seed=8)
    rig.load(0, p)
    how = dict(window="sliding", size=150)            # sees from 251 on: inside block 3
    page = int(rig.table[rig.slots[0], 3])
    rig.cache.v.view(torch.uint8)[page, :, :251 - 192] = 0x7f        # NaN
    rig.cache.k.view(torch.uint8)[page, :, :251 - 192] = 0xff
    rig.v[0][192:251] = 0
    rig.k[0][192:251] = 0
    q, out = rig.decode([p], **how)
    # (the reference holds block 3 as loaded: its visible rows decide the same scale, checked here)
    held = rig.cache.v[page].float() * rig.cache.v_scale[page][:, None, None]
    assert held[:, 251 - 192:].isfinite().all() and not out.isnan().any()
    rig2 = Rig([p + 1], fmt="e4m3", seed=8)
    rig2.load(0, p)
    _, out2 = rig2.decode([p], q=q, **how)
    assert torch.equal(out, out2)


def test_numbers_that_are_not_finite():
    """Held in 8 bits an infinity is the largest code, a NaN e4m3's NaN or int8's 0; neither enters the scale."""
    for fmt in ("int8", "e4m3"):
        rig = Rig([64], fmt=fmt, nh=2, nkv=1, d=64, seed=9)
        rig.k[0][3, 0, 5], rig.k[0][10, 0, 6], rig.v[0][7, 0, 8] = math.inf, -math.inf, math.nan
        rig.prompt([64])
        page = int(rig.table[rig.slots[0], 0])
        k, v = rig.cache.k[page, 0].float(), rig.cache.v[page, 0].float()
        most = 127.0 if fmt == "int8" else 448.0
        assert k[3, 5] == most and k[10, 6] == -most
        assert (v[7, 8] == 0.0) if fmt == "int8" else v[7, 8].isnan()
        rig.check_held(0)


# ---- prompts -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt,nh,nkv,d", [("int8", 4, 2, 128), ("e4m3", 5, 1, 64)])
@pytest.mark.parametrize("news", [[1, 2], [37], [63, 64, 65], [128, 129, 127], [255, 256, 257], [700, 33, 1, 260]])
def test_prompts(fmt, nh, nkv, d, news):
    rig = Rig([n + 1 for n in news], fmt=fmt, nh=nh, nkv=nkv, d=d, seed=len(news))
    q, out, _ = rig.prompt(news)
    for i, n in enumerate(news):
        some = sorted({0, 1, n // 3, n // 2, n - 2, n - 1, 63, 64, 65, 127, 128, 129, 191, 192, 255, 256} & set(range(n)))
        rig.check(i, q[i][some], out[i][some], some)
        rig.check_held(i)


@pytest.mark.parametrize("how", WINDOWS)
@pytest.mark.parametrize("pasts,news", [([70, 0, 128], [300, 140, 64]), ([257], [500])])
def test_later_pieces(how, pasts, news):
    """Pieces of prompts that start inside a block, at its end and at a border, under every window."""
    rig = Rig([p + n for p, n in zip(pasts, news)], nh=4, nkv=2, seed=11)
    for i, p in enumerate(pasts):
        rig.load(i, p)
    q, out, starts = rig.prompt(news, **how)
    for i, (s, n) in enumerate(zip(starts, news)):
        some = sorted({0, 1, 2, n // 4, n // 2, n - 1, (64 - s % 64) % 64, (63 - s % 64) % 64, 127, 128} & set(range(n)))
        rig.check(i, q[i][some], out[i][some], [s + x for x in some], **how)
        rig.check_held(i)


@pytest.mark.parametrize("nh,nkv,d,past,news", [(1, 1, 64, 3000, [2]), (2, 1, 128, 2111, [300]), (4, 4, 64, 5000, [130, 64]), (2, 2, 128, 1300, [1, 513])])
@pytest.mark.parametrize("how", [dict(), dict(window="sliding", size=1500, keep=70), dict(window="chunk", size=1000)])
def test_few_query_tiles_over_long_contexts(nh, nkv, d, past, news, how):
    """Few blocks of threads over many keys: a query tile's keys are shared out, with sinks and without."""
    rig = Rig([past + n for n in news], fmt="e4m3", nh=nh, nkv=nkv, d=d, seed=past)
    for i in range(len(news)):
        rig.load(i, past)
    sink = torch.linspace(-2, 6, nh, device=DEV) if nh > 2 else None
    q, out, starts = rig.prompt(news, sink=sink, **how)
    for i, (s, n) in enumerate(zip(starts, news)):
        some = sorted({0, 1, n // 2, n - 1, 63, 64, 127, 128, 255, 256} & set(range(n)))
        rig.check(i, q[i][some], out[i][some], [s + x for x in some], sink=sink, **how)
        rig.check_held(i)


@pytest.mark.parametrize("softcap", [0.0, 8.0])
def test_prompt_sink_and_cap(softcap):
    rig = Rig([300], nh=8, nkv=2, d=64, seed=12)
    sink = torch.tensor([-3.0, 0.0, 5.0, 200.0, -200.0, 1.0, 2.0, 3.0], device=DEV)
    q, out, _ = rig.prompt([300], sink=sink, softcap=softcap)
    some = [0, 1, 63, 64, 130, 299]
    rig.check(0, q[0][some], out[0][some], some, sink=sink, softcap=softcap)


@pytest.mark.parametrize("d,nkv", [(64, 1), (128, 2)])
@pytest.mark.parametrize("how", [dict(), dict(window="sliding", size=300, keep=3), dict(softcap=500.0)])
def test_scores_that_rise(d, nkv, how):
    """Scores that go up by more than 2^40 in weight again and again, at the first and last columns of tiles and of their parts,
    inside and outside of masked tiles: whatever was added up before is worth nothing then, and what follows is."""
    n, done = 700, 90
    rig = Rig([n], nh=2, nkv=nkv, d=d, seed=50)
    u = (torch.randint(0, 2, (d,), generator=rig.g, device=DEV) * 2 - 1).float()
    level = torch.randn(n, generator=rig.g, device=DEV)
    jumps = [0, 3, 31, 32, 33, 63, 64, 95, 127, 128, 129, 200, 255, 256, 300, 383, 400, 511, 512, 600, 650, 690]
    for i, at in enumerate(jumps):
        level[at] = 38.0 * (i + 1)                  # (38 log2 e = 55; up to 836, what the tolerance covers)
        if at + 1 not in jumps:
            level[at + 1] = level[at] - 1.0
    rig.k[0] = (level[:, None, None] * u * d ** -0.5 + 0.1 * torch.randn(n, nkv, d, generator=rig.g, device=DEV)).bfloat16()
    rig.rows = lambda *shape: u.bfloat16().expand(*shape).contiguous()
    rig.load(0, done)
    q, out, _ = rig.prompt([n - done], **how)
    rig.check(0, q[0], out[0], list(range(done, n)), **how)
    rig.done = [0]
    q, out, _ = rig.prompt([n], **how)
    rig.check(0, q[0], out[0], list(range(n)), **how)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_cuts_do_not_matter(fmt):
    """A sequence in one step, in pieces and token by token: the same cache bit for bit, the same outputs as the definition."""
    n = 300
    rigs = []
    for cuts in ([300], [100, 1, 90, 109], [64, 64, 172], [190] + [1] * 110):
        rig = Rig([n], fmt=fmt, nh=4, nkv=2, seed=13)
        for c in cuts:
            if c == 1:
                q, out = rig.decode([rig.done[0]])
                rig.check(0, q, out, [rig.done[0]])
                rig.done[0] += 1
            else:
                q, out, starts = rig.prompt([c])
                some = [0, c // 2, c - 1]
                rig.check(0, q[0][some], out[0][some], [starts[0] + x for x in some])
        rig.check_held(0)
        rigs.append(rig)


def test_slots_used_again():
    """A slot's next sequence finds the last one's tail and pages there and sees none of it."""
    rig = Rig([200, 90], seed=14)
    rig.prompt([200, 90])
    for i, n in enumerate((150, 80)):
        rig.k[i], rig.v[i] = rig.rows(n, 2, 128), rig.rows(n, 2, 128)
        rig.done[i] = 0
    q, out, _ = rig.prompt([150, 80])
    for i, n in enumerate((150, 80)):
        rig.check(i, q[i][[0, n - 1]], out[i][[0, n - 1]], [0, n - 1])
        rig.check_held(i)


# ---- how the calls behave ------------------------------------------------------------------------------------------
def test_captured_and_replayed_beside_an_eager_call():
    """Two captured graphs and an eager call, replayed on streams of their own at once: nothing is shared between them."""
    rigs = [Rig([3001], nh=8, nkv=1, seed=20 + i) for i in range(3)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)       # noqa: E731
    calls = []
    for rig in rigs:
        rig.load(0, 3000)
        rig.store_newest(0, 3000)
        q, out = rig.rows(1, 8 * 128), torch.zeros(1, 8 * 128, dtype=torch.bfloat16, device=DEV)
        index = (i32([0]), i32([3000]), i32(rig.slots))

        def call(rig=rig, q=q, out=out, index=index):
            K.attention_decode_kv8(q, out, rig.cache, rig.table, *index, n_heads=8, scale=128 ** -0.5, max_context=3001)
        calls.append((call, q, out))
    calls[0][0]()
    torch.cuda.synchronize()
    graphs = []
    for call, _, _ in calls[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call()
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            calls[2][0]()
    torch.cuda.synchronize()
    for rig, (_, q, out) in zip(rigs, calls):
        rig.check(0, q.view(1, 8, 128), out.view(1, 8, 128), [3000])


def test_a_sequence_that_is_not_finite_leaves_the_others_alone():
    """Sequences of one step lie side by side in the packed tokens and in the step's pages; what one holds reaches no other."""
    for fmt in ("int8", "e4m3"):
        rig = Rig([90, 70, 200], fmt=fmt, nh=4, nkv=2, d=64, seed=31)
        rig.k[1][3], rig.v[1][5], rig.v[1][69] = math.inf, math.nan, -math.inf
        q, out, _ = rig.prompt([90, 70, 200])
        assert out[1][69].isnan().any()
        for i, n in ((0, 90), (2, 200)):
            rig.check(i, q[i], out[i], list(range(n)))
            rig.check_held(i)


def test_prompts_at_once():
    """Prompts of two caches on two streams, again and again: nothing is shared between the calls."""
    news, done = [300, 65], []
    rigs = [Rig(news, nh=4, nkv=2, seed=40 + i) for i in range(2)]
    for rig in rigs:                                # what a prompt alone gives
        q, out, _ = rig.prompt(news)
        for i, n in enumerate(news):
            rig.check(i, q[i], out[i], list(range(n)))
        batch = rig.stager.stage(rig.slots, [0, 0], [[0] * m for m in news], [[]] * 2, torch.bfloat16)
        plan = Kv8Plan([0, 0], news, rig.slots, device=DEV)
        pages = [torch.zeros(plan.n_pages, 2, BLOCK, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
        at, row = plan.exact_table.long()[batch.token_seq.long(), (batch.token_pos // BLOCK).long()], (batch.token_pos % BLOCK).long()
        for to, x in zip(pages, (rig.k, rig.v)):
            to[at, :, row] = torch.cat(x)
        done.append((rig, torch.cat(q).view(sum(news), -1), torch.cat(out).view(sum(news), -1), plan, batch, pages))
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(5):
        for s, (rig, q, _, plan, batch, pages) in zip(streams, done):
            with torch.cuda.stream(s):
                out = torch.zeros_like(q)
                K.kv8_stage(rig.cache, rig.table, plan, *pages)
                K.attention_prefill_kv8(q, out, *pages, plan, batch.token_seq, batch.token_pos, batch.tile_tok0, batch.tile_rows, n_heads=4,
                                        scale=128 ** -0.5)
                outs.append(out)
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        assert torch.equal(out, done[i % 2][2])


def test_same_results_twice():
    rig = Rig([2000, 77], nh=8, nkv=2, seed=25)
    for i, p in enumerate((1999, 76)):
        rig.load(i, p)
    q, a = rig.decode([1999, 76])
    _, b = rig.decode([1999, 76], q=q)
    assert torch.equal(a, b)
