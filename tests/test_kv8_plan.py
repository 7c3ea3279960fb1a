"""The plan of a step on the cache in 8 bits, and the refusals of its calls and of `log_probs` (no device needed)."""
from __future__ import annotations

import random
import re
from types import SimpleNamespace

import pytest
import torch

import kv8_plain as P
from cpi_b200.cache.kv8 import Kv8Cache, Kv8Plan, needed_blocks
from cpi_b200.cache.manager import KVRequirement
from cpi_b200.csrc import lib as K
from test_kernel_order import KERNELS


def draws(n):
    rng = random.Random(3)
    for _ in range(n):
        window = rng.choice(["full", "chunk", "sliding"])
        size = 0 if window == "full" else rng.choice([1, 30, 64, 100, 128, 300])
        keep = rng.choice([0, 3, 64, 130]) if window == "sliding" else 0
        m = rng.randint(1, 4)
        starts = [rng.choice([0, 63, 64, 65, rng.randrange(700)]) for _ in range(m)]
        news = [rng.choice([1, 2, 63, 64, 65, rng.randrange(1, 400)]) for _ in range(m)]
        yield window, size, keep, starts, news, rng.sample(range(9), m)


@pytest.mark.parametrize("case", list(draws(60)))
def test_every_block_that_a_token_sees_has_a_page(case):
    window, size, keep, starts, news, slots = case
    plan = Kv8Plan(starts, news, slots, window_kind=window, window_size=size, keep_first=keep, device="cpu")
    assert plan.n_tokens == sum(news) and plan.jobs.numel() == 8 * plan.n_jobs
    used = []
    jobs = plan.jobs.view(-1, 8).tolist()
    for i, (s, n) in enumerate(zip(starts, news)):
        earlier = {b for p in range(s, s + n) for b in {r // 64 for r in P.rows_seen(p, window, size, keep)} if b < p // 64}
        have = {b for b in range(plan.width) if int(plan.earlier_table[i, b]) >= 0}
        assert earlier <= have and have <= set(range((s + n - 1) // 64))
        assert have == set(needed_blocks(s, n, window, size, keep))
        own = {b for b in range(plan.width) if int(plan.exact_table[i, b]) >= 0}
        assert own == set(range(s // 64, (s + n - 1) // 64 + 1))
        used += [int(plan.earlier_table[i, b]) for b in have] + [int(plan.exact_table[i, b]) for b in own]
        mine = [j for j in jobs if j[0] == slots[i]]
        # a job per own block and one per earlier block that was complete before; completed ones are written by their own
        assert sorted(j[1] for j in mine if j[5] >= 0) == sorted(own)
        assert sorted(j[1] for j in mine if j[5] < 0) == sorted(b for b in have if b < s // 64)
        for slot, b, r0, rows, page, exact, last, last_rows in mine:
            assert page == int(plan.earlier_table[i, b])
            if exact >= 0:
                assert exact == int(plan.exact_table[i, b])
                assert r0 == (s - b * 64 if b == s // 64 else 0) and rows == min(64, s + n - b * 64)
                assert (last >= 0) == (b == s // 64)
                if last >= 0:
                    assert last == int(plan.exact_table[i, (s + n - 1) // 64]) and last_rows == (s + n - 1) % 64 + 1
    assert sorted(used) == list(range(plan.n_pages))
    assert all(int(x) < plan.n_earlier for x in plan.earlier_table.flatten()) and all(j[5] < 0 or j[5] >= plan.n_earlier for j in jobs)


@pytest.mark.parametrize("case", list(draws(40)))
def test_the_cache_still_holds_what_a_step_needs(case):
    """Pages that a window has let go of at the start of a step are not asked for by it."""
    window, size, keep, starts, news, _ = case
    req = KVRequirement(1, 64, window, size, keep_first=keep)
    for s, n in zip(starts, news):
        for b in needed_blocks(s, n, window, size, keep):
            assert not req.droppable(b, s, 64)


@pytest.mark.parametrize("bad", [dict(window_kind=5), dict(window_kind=1, window_size=0), dict(window_kind=2, window_size=1 << 40), dict(keep_first=-1),
                                 dict(scale=0.0), dict(scale=float("nan")), dict(softcap=-1.0), dict(softcap=float("nan")), dict(sink=torch.zeros(3)),
                                 dict(sink=torch.zeros(4, dtype=torch.float64))])
def test_options_refused(bad):
    good = dict(scale=1.0, window_kind=0, window_size=0, keep_first=0, sink=None, softcap=0.0)
    K._attention_options("test", 4, *good.values())
    with pytest.raises(K.KernelError):
        K._attention_options("test", 4, *{**good, **bad}.values())


def test_plan_refusals():
    good = dict(starts=[0], n_new=[1], slots=[0], device="cpu")
    Kv8Plan(**good)
    for change in (dict(starts=[0, 1]), dict(n_new=[0]), dict(starts=[-1]), dict(slots=[-2]), dict(window_kind="round"),
                   dict(window_kind="chunk"), dict(starts=[], n_new=[], slots=[]), dict(starts=[0, 0], n_new=[1, 1], slots=[3, 3])):
        with pytest.raises(ValueError):
            Kv8Plan(**{**good, **change})


def cpu_cache(pages=2, nkv=2, d=64, kind=torch.int8, slots=1, block=64):
    z = lambda *s, t: torch.zeros(*s).to(t)       # noqa: E731
    return Kv8Cache(z(pages, nkv, block, d, t=kind), z(pages, nkv, block, d, t=kind), z(pages, nkv, t=torch.float32),
                    z(pages, nkv, t=torch.float32), z(slots, nkv, block, d, t=torch.bfloat16), z(slots, nkv, block, d, t=torch.bfloat16))


@pytest.mark.parametrize("change", [
    dict(k=torch.zeros(2, 2, 64, 64)), dict(k=torch.zeros(2, 2, 64, 32, dtype=torch.int8)), dict(v=torch.zeros(3, 2, 64, 64, dtype=torch.int8)),
    dict(k_scale=torch.zeros(2, 3)), dict(v_scale=torch.zeros(2, 2, dtype=torch.float64)), dict(k_tail=torch.zeros(1, 2, 64, 64)),
    dict(v_tail=torch.zeros(2, 2, 64, 64).bfloat16()), dict(k_scale=torch.zeros(2, 4)[:, ::2])])
def test_cache_refusals(change):
    with pytest.raises(K.KernelError):
        K._kv8(cpu_cache()._replace(**change), "test")


@pytest.mark.parametrize("bad", [dict(nkv=2, n_heads=3), dict(nkv=1, n_heads=17), dict(nkv=2, n_heads=0), dict(block=32), dict(d=96)])
def test_shapes_refused(bad):
    heads = bad.pop("n_heads", None)
    with pytest.raises(K.KernelError):
        K._kv8(cpu_cache(**bad), "test", heads)


def test_calls_refuse_the_host():
    """There is no CPU path: tensors of the host are refused before anything is launched."""
    c = cpu_cache()
    i = torch.zeros(1, dtype=torch.int32)
    q = torch.zeros(1, 128).bfloat16()
    with pytest.raises(K.KernelError, match="CUDA"):
        K.attention_decode_kv8(q, q.clone(), c, i.view(1, 1), i, i, i, n_heads=2, scale=1.0, max_context=1)
    plan = Kv8Plan([0], [1], [0], device="cpu")
    pages = torch.zeros(1, 2, 64, 64).bfloat16()
    with pytest.raises(K.KernelError, match="CUDA"):
        K.kv8_stage(c, i.view(1, 1), plan, pages, pages.clone())
    with pytest.raises(K.KernelError, match="CUDA"):
        K.attention_prefill_kv8(q, q.clone(), pages, pages.clone(), plan, i, i, i, i, n_heads=2, scale=1.0)
    with pytest.raises(K.KernelError, match="CUDA"):
        K.log_probs(torch.zeros(1, 5), i)


@pytest.mark.parametrize("logits,targets,top", [
    (torch.zeros(5), torch.zeros(5, dtype=torch.int32), 0), (torch.zeros(2, 5, dtype=torch.float16), torch.zeros(2, dtype=torch.int32), 0),
    (torch.zeros(2, 5), torch.zeros(3, dtype=torch.int32), 0), (torch.zeros(2, 5), torch.zeros(2), 0), (torch.zeros(2, 0), torch.zeros(2, dtype=torch.int32), 0),
    (torch.zeros(2, 5), torch.zeros(2, dtype=torch.int32), 6), (torch.zeros(2, 50), torch.zeros(2, dtype=torch.int32), 33),
    (torch.zeros(2, 5), torch.zeros(2, dtype=torch.int32), -1), (torch.zeros(5, 2).t(), torch.zeros(2, dtype=torch.int32), 0),
    (torch.zeros(2, 5), torch.zeros(3, 2, dtype=torch.int32).t(), 0)])
def test_log_probs_refusals(logits, targets, top):
    with pytest.raises(K.KernelError):
        K.log_probs(logits, targets, top=top)


def test_arguments_are_declared_as_the_library_has_them():
    """The kinds that a binding declares are those of the C function, one for one."""
    import os
    import re
    folder = os.path.dirname(K.__file__)
    sources = "".join(open(os.path.join(folder, f)).read() for f in sorted(os.listdir(folder)) if f.endswith(".cu"))
    declared = re.findall(r'_declared\("(\w+)", "(\w+)"\)', open(K.__file__).read())
    assert len(declared) >= 4
    for name, types in declared:
        args = re.search(r'extern "C" int ' + name + r"\(([^)]*)\)", sources).group(1).split(",")
        kinds = ["p" if "*" in a or "cudaStream_t" in a else "f" if "float " in a else "l" if "long " in a else "i" for a in args]
        assert "".join(kinds) == types, name


@pytest.mark.parametrize("name", ["attention_decode_kv8.cu:attention_decode_kv8_kernel", "attention_prefill_kv8.cu:attention_prefill_kv8_kernel",
                                  "kv8_stage.cu:kv8_stage_kernel", "log_probs.cu:log_probs_kernel",
                                  "attention_decode_kv8.cu:attention_decode_kv8_combine", "attention_prefill_kv8.cu:attention_prefill_combine"])
def test_kernels_wait_before_they_read_and_before_their_successors_start(name):
    """Indices, codes, tails and logits may come from the kernel in front: nothing is read through a pointer before the wait, and
    successors, whose predecessors have to have stored their rows, start after it."""
    body = KERNELS[name]
    before = body[:body.index("pdl_wait()")]
    assert not re.search(r"\bp\.\w+\s*\[|\bpart_\w+\s*\[|tma_load|\bjob\s*\[|__ldcg|\*reinterpret_cast", before)
    assert all(body.index("pdl_wait()") < m.start() for m in re.finditer(r"pdl_launch_dependents\(\)", body))


@pytest.mark.parametrize("tokens", [[], [3], [1, 50], [1, -1], [1, 2 ** 31], [2 ** 40, 1]])
def test_sequences_that_are_not_scored(tokens):
    from cpi_b200.engine.score import score_sequence
    engine = SimpleNamespace(spec=SimpleNamespace(vocab_size=50), max_step_tokens=8, device="cpu")
    with pytest.raises(ValueError):
        score_sequence(engine, tokens)


@pytest.mark.parametrize("argv", [["--interactive", "--logprobs", "2"], ["--interactive", "--score"], ["--score", "--benchmark"],
                                  ["--score", "--dump-logits", "x"], ["--logprobs", "33"], ["--logprobs", "-1"],
                                  ["--cache-dtype", "int8", "--dtype", "float32"]])
def test_options_of_the_command_line_that_do_not_go_together(argv, capsys):
    from cpi_b200.cli import llama_infer as cli
    assert cli.main(["m", *argv]) == 1
    assert argv[0] in capsys.readouterr().err
