"""Models whose attention layers keep their keys and values in 8 bits, and scores of tokens, through the public entry points."""
from __future__ import annotations

import json
import math
import os
import subprocess
import sys

import pytest
import torch

import kv8_plain as P
import nekorax_tiny
import savenex_tiny
import tiny
from cpi_b200.api import Model
from cpi_b200.csrc import lib as K
from cpi_b200.engine import Engine, StepEntry
from cpi_b200.engine import score as score_module

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# chunked and full layers, query temperature, heads of 128 in a group of four; no experts (a near tie of two experts would
# make two correct runs differ)
DENSE = {"architectures": ["Llama4ForCausalLM"], "num_hidden_layers": 4, "hidden_size": 256, "num_attention_heads": 8,
         "num_key_value_heads": 2, "head_dim": 128, "intermediate_size": 512, "intermediate_size_mlp": 512, "num_local_experts": 1,
         "num_experts_per_tok": 1, "interleave_moe_layer_step": 1 << 20, "vocab_size": 777, "rms_norm_eps": 1e-5, "rope_theta": 5e5,
         "nope_layer_interval": 2, "attention_chunk_size": 160, "use_qk_norm": True, "attn_temperature_tuning": True, "floor_scale": 100,
         "attn_scale": 0.2, "tie_word_embeddings": False, "max_position_embeddings": 4096, "initializer_range": 0.05}
# attention beside a recurrence: windows with kept first positions, everything visible
BESIDE = savenex_tiny.model([
    savenex_tiny.layer(savenex_tiny.left(4, 1, 64, 64, window=40, keep_first=5, rot_dims=64), savenex_tiny.right(4, 2, 64, 64, 4),
                       savenex_tiny.dense(192, 3.0)),
    savenex_tiny.layer(savenex_tiny.left(4, 2, 128, 128, window=150, keep_first=70, rot_dims=64), savenex_tiny.right(2, 2, 48, 64, 3),
                       savenex_tiny.dense(64, 3.0)),
    savenex_tiny.layer(savenex_tiny.left(2, 2, 64, 64, rot_dims=16), savenex_tiny.right(8, 4, 16, 32, 2), None)],
    width=128, vocab=384, loop=(1, 2, 2))
# short convolutions, values that turn, a sink and gates, beside layers of another kind that keep what they keep
TURNED = nekorax_tiny.model([
    nekorax_tiny.layer(nekorax_tiny.attention(4, 2, 64, 64, 32, conv=4), None),
    nekorax_tiny.layer(nekorax_tiny.latent(4, 32, 16, 48, 48, 96, window=50), None),
    nekorax_tiny.layer(nekorax_tiny.attention(6, 1, 128, 128, 128), None)], width=192, vocab=384)
CONFIGS = {"dense": DENSE, "beside": BESIDE, "turned": TURNED}
_engines = {}


def engine(name, held, **kw):
    key = (name, held, tuple(kw.items()))
    if key not in _engines:
        _engines[key] = Engine.from_random(CONFIGS[name], 3, dtype="bfloat16", max_tokens=4096, max_seqs=4, max_seq_len=1024, cache_dtype=held, **kw)
    assert not _engines[key].cache.live_slots()
    return _engines[key]


def vocab(name):
    return CONFIGS[name].get("vocab_size") or CONFIGS[name]["vocab"]


def run(e, seqs, cuts):
    """Logits of every position of each sequence, run side by side in steps of cuts[i] tokens."""
    slots = [e.acquire_slot() for _ in seqs]
    rows = [[] for _ in seqs]
    at = [0] * len(seqs)
    for step in cuts:
        entries, who = [], []
        for i, (s, toks) in enumerate(zip(slots, seqs)):
            n = min(step, len(toks) - at[i])
            if n > 0:
                entries.append(StepEntry(s, toks[at[i]:at[i] + n], range(n)))
                who.append((i, n))
                at[i] += n
        if entries:
            logits = e.step(entries)
            for (i, _), part in zip(who, logits.split([n for _, n in who])):
                rows[i].append(part.clone())
    e.check_device_errors()
    for s in slots:
        e.release_slot(s)
    e.cache.check_consistency()
    assert at == [len(t) for t in seqs]
    return [torch.cat(r) for r in rows]


class Watch:
    """Records what every layer's attention was given and what it answered, step by step (eager steps only)."""

    def __init__(self, monkeypatch, e):
        self.calls, self.e = [], e
        stage, prefill, decode = K.kv8_stage, K.attention_prefill_kv8, K.attention_decode_kv8

        def watched_stage(cache, table, plan, k_pages, v_pages):
            self.rows = (plan, k_pages.clone(), v_pages.clone())        # the exact pages hold the step's rows, as projected
            stage(cache, table, plan, k_pages, v_pages)

        def watched_prefill(q, out, k_pages, v_pages, plan, token_seq, token_pos, *a, **how):
            prefill(q, out, k_pages, v_pages, plan, token_seq, token_pos, *a, **how)
            page = plan.exact_table.long()[token_seq.long(), (token_pos // 64).long()]
            row = (token_pos % 64).long()
            assert self.rows[0] is plan
            self.calls.append((q.clone(), out.clone(), self.rows[1][page, :, row], self.rows[2][page, :, row], token_seq.tolist(),
                               token_pos.tolist(), how))

        def watched_decode(q, out, cache, table, token_seq, token_pos, seq_slot, **how):
            slot, row = seq_slot[token_seq.long()].long(), (token_pos % 64).long()
            k, v = cache.k_tail[slot, :, row].clone(), cache.v_tail[slot, :, row].clone()
            decode(q, out, cache, table, token_seq, token_pos, seq_slot, **how)
            self.calls.append((q.clone(), out.clone(), k, v, token_seq.tolist(), token_pos.tolist(), how))

        monkeypatch.setattr(K, "kv8_stage", watched_stage)
        monkeypatch.setattr(K, "attention_prefill_kv8", watched_prefill)
        monkeypatch.setattr(K, "attention_decode_kv8", watched_decode)


@pytest.mark.parametrize("held", ["int8", "e4m3"])
@pytest.mark.parametrize("name", sorted(CONFIGS))
def test_every_layers_attention(name, held, monkeypatch):
    """In a model, whatever the cuts: each layer's outputs are those of the definition on the rows that its projections made."""
    e = engine(name, held)
    seqs = [tiny.random_tokens(n, vocab(name), n) for n in (300, 129, 64, 5)]
    window_of = {v: k for k, v in K.WINDOW_KINDS.items()}
    monkeypatch.setattr(e, "use_graphs", False)
    for cuts in ([1000], [100, 1, 1, 60, 300], [190] + [1] * 110, [64, 64, 63, 1, 300]):
        with monkeypatch.context() as m:
            watch = Watch(m, e)
            run(e, seqs, cuts)
        steps = sum(any(sum(cuts[:i]) < len(t) for t in seqs) for i in range(len(cuts)))
        layers = len(watch.calls) // steps
        assert layers * steps == len(watch.calls) and layers >= 2
        for layer in range(layers):
            k, v, live = {}, {}, []
            for q, out, kr, vr, who, pos, how in watch.calls[layer::layers]:
                n = max(who) + 1
                if not live:
                    live = list(range(len(seqs)))
                # (a sequence that is through has left the step; the others keep their order)
                live = [i for i in live if len(k.get(i, ())) < len(seqs[i])]
                assert n == len(live)
                for t, (s, p) in enumerate(zip(who, pos)):
                    i = live[s]
                    assert len(k.setdefault(i, [])) == p
                    k[i].append(kr[t])
                    v.setdefault(i, []).append(vr[t])
                for s in range(n):
                    i = live[s]
                    mine = [t for t in range(len(who)) if who[t] == s]
                    some = [t for t in mine if pos[t] % 64 in (0, 17, 63) or t == mine[-1]]
                    if len(mine) == 1 and pos[mine[0]] % 16 not in (0, 15):
                        continue
                    heads = how["n_heads"]
                    d = q.shape[1] // heads
                    ref, mag = P.attend(q[some].view(-1, heads, d), torch.stack(k[i]), torch.stack(v[i]), [pos[t] for t in some], fmt=held,
                                        scale=how["scale"], window=window_of[how["window_kind"]], size=how["window_size"],
                                        keep=how["keep_first"], sink=how["sink"], softcap=how["softcap"])
                    err = (out[some].view(-1, heads, d).double() - ref).abs()
                    assert bool((err <= P.tolerance(ref, mag)).all()), f"layer {layer} sequence {i} cuts {cuts[:5]}: {float(err.max())}"


@pytest.mark.parametrize("name", sorted(CONFIGS))
def test_replayed_steps_are_eager_steps(name, monkeypatch):
    """Decode steps through captured graphs give the bits of the same steps launched one by one."""
    e = engine(name, "int8")
    assert e.use_graphs
    seqs = [tiny.random_tokens(n, vocab(name), n) for n in (180, 130)]
    cuts = [100] + [1] * 80
    replayed = run(e, seqs, cuts)
    monkeypatch.setattr(e, "use_graphs", False)
    for a, b in zip(replayed, run(e, seqs, cuts)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("name", sorted(CONFIGS))
def test_cuts_do_not_matter(name):
    """A query's own block is exact and earlier ones are held in 8 bits whatever step brought them.  Two cuts project rows by
    products of other shapes, which agree to bfloat16 (half a step: 2^-8); where such a difference crosses the border of
    two int8 codes, the held numbers are a step apart, up to 2 max / 127 = 2^-6 of the block's largest: four times
    as much.  So the logits agree to four times what they do without 8 bits (2e-2 of the largest)."""
    e = engine(name, "int8")
    seqs = [tiny.random_tokens(n, vocab(name), n) for n in (330, 129, 64, 5)]
    whole = run(e, seqs, [1000])
    for cuts in ([100, 1, 1, 60, 300], [190] + [1] * 140, [64, 64, 63, 1, 300]):
        for a, b in zip(whole, run(e, seqs, cuts)):
            assert float((a - b).abs().max()) <= 4 * 2e-2 * float(a.abs().max()), f"cuts {cuts[:5]}"


@pytest.mark.parametrize("held,most", [("int8", 0.05), ("e4m3", 0.1)])
@pytest.mark.parametrize("name", sorted(CONFIGS))
def test_near_the_model_without_8_bits(name, held, most):
    """The first block is exact; later logits are off by what 8 bits take, in the mean.  int8 codes are off by up to max / 127, a
    third of that rms with the largest of a block near 4 sigma: 2% of a number; e4m3 by 2^-4 / sqrt(3) = 4%; twice that for
    what keys and values do together."""
    seqs = [tiny.random_tokens(400, vocab(name), 1)]
    plain, = run(engine(name, None), seqs, [1000])
    got, = run(engine(name, held), seqs, [1000])
    scale = plain.std()
    assert float((plain[:64] - got[:64]).abs().max()) <= 2e-2 * float(plain.abs().max())
    off = float((plain[64:] - got[64:]).std() / scale)
    assert 0.0 < off < most


def test_slots_and_pages_used_again():
    """More requests than slots, in a cache that holds two of them: later ones find nothing of earlier ones."""
    m = Model(engine("dense", "int8"), 4)
    prompts = [tiny.random_tokens(n, 777, n) for n in (70, 200, 64, 127, 128, 3, 190)]
    together = m.generate(prompts, max_new=80, temperature=0.0, stop_ids=[])
    for p, r in zip(prompts, together):
        alone = m.generate([p], max_new=80, temperature=0.0, stop_ids=[], logprobs=2)[0]
        for a, b, s in zip(r.tokens, alone.tokens, alone.scores):
            if a != b:                       # a near tie of the two best tokens may fall either way
                assert s.top[0][1] - s.top[1][1] < 0.1
                break


def test_scores_are_the_steps_logits():
    """`score`, a prompt's logits and log_softmax in 64 bits; in one piece and in several."""
    for held in (None, "int8"):
        e = engine("dense", held)
        m = Model(e, 4)
        seqs = [tiny.random_tokens(n, 777, n + 7) for n in (2, 65, 300)]
        got = m.score(seqs, top=3)
        kept = score_module.LOGIT_BYTES
        score_module.LOGIT_BYTES = 4 * 777 * 50
        try:
            pieces = m.score(seqs, top=3)
        finally:
            score_module.LOGIT_BYTES = kept
        for toks, a, b in zip(seqs, got, pieces):
            assert len(a) == len(b) == len(toks) - 1
            logits, = run(e, [toks], [1000])
            lp = torch.log_softmax(logits[:-1].double(), -1)
            for i, (x, y) in enumerate(zip(a, b)):
                # (one piece: the same logits, so float32 rounding only; several: other shapes of the same products)
                assert abs(x.logprob - float(lp[i, toks[i + 1]])) < 1e-4
                assert abs(x.entropy - float(-(lp[i].exp() * lp[i]).sum())) < 1e-4
                assert [t for t, _ in x.top] == torch.sort(logits[i], descending=True, stable=True).indices[:3].tolist()
                assert abs(x.logprob - y.logprob) < 2e-2 * float(logits.abs().max()) * 2
    with pytest.raises(ValueError):
        m.score([[5]])
    with pytest.raises(ValueError):
        m.score([[5, 777]])
    assert not e.cache.live_slots()


def test_generated_tokens_with_their_scores():
    m = Model(engine("dense", "e4m3"), 4)
    prompts = [tiny.random_tokens(n, 777, n) for n in (5, 70)]
    plain = m.generate(prompts, max_new=8, temperature=0.0, stop_ids=[])
    scored = m.generate(prompts, max_new=8, temperature=0.0, stop_ids=[], logprobs=4)
    assert all(r.scores is None for r in plain)
    for a, b in zip(plain, scored):
        assert a.tokens == b.tokens and len(b.scores) == 8
        for t, s in zip(b.tokens, b.scores):
            assert len(s.top) == 4 and s.top[0][0] == t and s.top[0][1] == s.logprob and 0 < s.entropy < math.log(777)
    for p, r in zip(prompts, m.generate(prompts, max_new=6, temperature=1.0, repetition_penalty=1.3, seed=5, stop_ids=[], logprobs=0)):
        assert len(r.scores) == 6 and all(s.top == [] for s in r.scores)
        again = m.score([p + r.tokens])[0][-6:]       # the model's own distribution, not the penalised one
        for s, t in zip(r.scores, again):
            assert abs(s.logprob - t.logprob) < 0.2
    with pytest.raises(ValueError):
        m.generate(prompts, logprobs=-1)


def test_command_line(tmp_path):
    cfg = tmp_path / "config.json"
    cfg.write_text(json.dumps(DENSE))
    env = {**os.environ, "LLAMA_INFER_LOCK_PATH": str(tmp_path / "lock")}
    base = [sys.executable, os.path.join(ROOT, "bin", "llama_infer"), "--random", str(cfg), "--tokens", "5,6,7,8", "--max-new", "3", "--temp",
            "0", "--eos-token", "-1", "--max-context", "256"]
    out = subprocess.run(base + ["--cache-dtype", "int8", "--logprobs", "2"], capture_output=True, text=True, env=env, timeout=300)
    assert out.returncode == 0, out.stderr
    lines = [x for x in out.stdout.splitlines() if x.startswith("  id=")]
    assert len(lines) == 3 and all("logprob=" in x and x.count(":") == 2 for x in lines)
    out = subprocess.run(base + ["--score"], capture_output=True, text=True, env=env, timeout=300)
    assert out.returncode == 0 and "[score] prompt=0 tokens=3 " in out.stdout and "Output tokens" not in out.stdout


def test_refusals():
    for kw in (dict(cache_dtype="int4"), dict(cache_dtype="int8", dtype="float32"), dict(cache_dtype="int8", page_size=32)):
        with pytest.raises(ValueError):
            Engine.from_random(DENSE, 0, **{"dtype": "bfloat16", "max_tokens": 256, **kw})
    small = {**DENSE, "head_dim": 32}
    with pytest.raises(ValueError, match="8 bits"):
        Engine.from_random(small, 0, dtype="bfloat16", max_tokens=256, cache_dtype="int8")
    latent = nekorax_tiny.model([nekorax_tiny.layer(nekorax_tiny.latent(4, 32, 16, 48, 48, 96), None)], width=192, vocab=384)
    with pytest.raises(ValueError, match="no layer"):
        Engine.from_random(latent, 0, dtype="bfloat16", max_tokens=256, cache_dtype="e4m3")
