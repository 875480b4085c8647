"""Several answers to many prompts: how often a prompt is computed, what they are, and which calls are refused before anything runs."""

from __future__ import annotations

import pytest
import torch

from harness import TinyEngine, random_prompt
from mini_llm_runtime_b200 import ops
from mini_llm_runtime_b200.ops import cuda_ops
from requests_support import RequestFakeOps
from test_shared_pages_cpu import SharedFakeOps
from test_forked_requests_cpu import engine_of, rows_run
from tiny_configs import TINY

LIMITS = {"temperature": 1.5, "top_k": 20}


class Kernels(RequestFakeOps, SharedFakeOps):
    def __init__(self):
        RequestFakeOps.__init__(self)
        SharedFakeOps.__init__(self)


@pytest.fixture(autouse=True)
def kernels(monkeypatch):
    monkeypatch.setattr(cuda_ops, "_need", lambda *args, **kwargs: None)
    with ops.use(Kernels()) as stand_in:
        yield stand_in


@pytest.fixture
def tiny():
    return TinyEngine(*TINY["A"], torch.float32, "cpu")


def by_themselves(tiny, prompts, answers, count, seed, **options):
    want = []
    for i, prompt in enumerate(prompts):
        for j in range(answers):
            want += engine_of(tiny, sampling_limits=True).generate([prompt], max_new_tokens=count, seed=seed + answers * i + j, **options)
    return want


@pytest.mark.parametrize("slots,answers", [(2, 3), (4, 2), (4, 3), (3, 5)])
@pytest.mark.parametrize("step_ahead", [False, True])
def test_a_prompt_is_computed_once_with_more_prompts_than_slots(slots, answers, step_ahead, tiny, monkeypatch):
    prompts = [random_prompt(tiny.config.vocab_size, n, n) for n in (19, 5, 33, 16, 8)]
    engine = engine_of(tiny, sampling_limits=True, max_running_requests=slots, total_blocks=60, step_ahead=step_ahead)
    rows, asked, step = [], {}, engine.runner.step
    count = 4

    def noted(entries, **kw):
        for entry in entries:
            asked[entry.request_id] = asked.get(entry.request_id, 0) + len(entry.tokens)
        return step(entries, **kw)

    monkeypatch.setattr(engine.runner, "step", noted)
    got = engine.generate(prompts, max_new_tokens=count, seed=3, answers=answers, **LIMITS)
    # each prompt once, its last token for each further answer, count - 1 tokens fed back each
    once = sum(len(p) for p in prompts) + len(prompts) * ((answers - 1) + answers * (count - 1))
    if slots % answers == 0 or slots < answers:
        assert sum(asked.values()) == once
    else:      # a first answer that got the place left over may have ended when the others' turn comes
        assert once <= sum(asked.values()) < answers * (sum(len(p) for p in prompts) + len(prompts) * (count - 1))
    assert got == by_themselves(tiny, prompts, answers, count, 3, **LIMITS)
    engine.manager.check_consistency()
    assert engine.manager.stats().free_pages == (60,) and engine.manager.stats().promised_pages == (0,)


@pytest.mark.parametrize("slots,count", [(1, 3), (4, 1)])
def test_answers_that_cannot_run_together_are_those_of_requests_by_themselves(slots, count, tiny):
    prompts = [random_prompt(tiny.config.vocab_size, n, n) for n in (9, 17)]
    engine = engine_of(tiny, sampling_limits=True, max_running_requests=slots)
    assert engine.generate(prompts, max_new_tokens=count, seed=3, answers=3, **LIMITS) == by_themselves(tiny, prompts, 3, count, 3, **LIMITS)


def test_a_fork_takes_the_place_of_the_request_that_it_began_as(tiny, monkeypatch):
    """Requests that wait until their parent has ended start with what the parent's other forks hold, each of them ending in its turn."""
    engine = engine_of(tiny, max_running_requests=2)
    prompt = random_prompt(tiny.config.vocab_size, 40, 1)
    engine.submit("a", prompt, max_new_tokens=3)
    engine.step()
    for i in range(4):
        engine.submit(f"f{i}", prompt[:30 + 3 * i], max_new_tokens=4, fork_of="a")
    rows = rows_run(engine, monkeypatch)
    engine.run()
    # f0 begins with 29 of a's tokens beside a, whose last two it outlives; f1 with 32 of its 33 while a runs, or else f0's 29, and so on
    assert sum(rows) <= 2 + sum((30 + 3 * i) - 29 + 3 for i in range(4))
    engine.manager.check_consistency()
    whole = engine_of(tiny)
    for i in range(4):
        assert list(engine.scheduler.get_request(f"f{i}").generated_token_ids) == whole.generate([prompt[:30 + 3 * i]], max_new_tokens=4)[0]


def test_answers_to_prompts_that_start_with_a_prefix(tiny, monkeypatch):
    page = TINY["A"][1]
    tokens = random_prompt(tiny.config.vocab_size, 2 * page, 1)
    prompt = tokens + random_prompt(tiny.config.vocab_size, 11, 2)
    want = by_themselves(tiny, [prompt], 3, 4, 5, **LIMITS)
    # with room for a request of its own pages the others fork; with room only beside the prefix's they share that
    for blocks, computed in ((40, 11 + 2), (5, 11 + 2), (4, 3 * 11)):      # 46 tokens, pages of 16
        engine = engine_of(tiny, sampling_limits=True, max_prefixes=1, total_blocks=blocks)
        engine.add_prefix("p", tokens)
        rows = rows_run(engine, monkeypatch)
        assert engine.generate([prompt], max_new_tokens=4, seed=5, answers=3, prefix="p", **LIMITS) == want
        assert sum(rows) == computed + 3 * 3
        engine.drop_prefix("p")
        assert engine.manager.stats().free_pages == (blocks,)


def test_a_prompt_that_is_refused_is_refused_before_any_runs(tiny, monkeypatch):
    engine = engine_of(tiny, sampling_limits=True)
    rows = rows_run(engine, monkeypatch)
    good = random_prompt(tiny.config.vocab_size, 9, 4)
    for bad, options in (([], {}), ([tiny.config.vocab_size], {}), (good * 30, {}), (good, {"max_new_tokens": 0}), (good, {"top_k": -1}),
                         (good, {"prefix": "p"}), (good, {"eos_token_ids": ["x"]})):
        with pytest.raises(ValueError):
            engine.generate([good, bad], **{"max_new_tokens": 2, "answers": 2, **options})
    assert rows == [] and not engine.scheduler.has_unfinished_requests
