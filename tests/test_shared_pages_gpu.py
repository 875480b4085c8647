"""Requests that start with another's pages, on the device: logits of decode steps through the attention of shared prefixes, eager and
captured, while the members of the groups change; the engine with prefixes, rules and steps ahead."""

from __future__ import annotations

import dataclasses

import pytest
import torch

from harness import TinyEngine, assert_close, random_prompt
from mini_llm_runtime_b200 import ops
from mini_llm_runtime_b200.engine import ContinuousBatchEngine, StepEntry
from tiny_configs import TINY

pytestmark = pytest.mark.gpu

CONFIGS = {"D": (dataclasses.replace(TINY["D"][0], use_sliding_window=False), TINY["D"][1]), "E": TINY["E"]}


@pytest.fixture
def shared_calls(monkeypatch):
    """Every prefix counts as worth its own walk; the calls of the shared attention's kernels."""
    kernels = ops.current()
    monkeypatch.setattr(kernels, "shared_prefix_least", 0)
    calls = []
    shared = kernels.shared_prefix_attention
    monkeypatch.setattr(kernels, "shared_prefix_attention", lambda *args: calls.append(args[4].counts["tile_keys"]) or shared(*args))
    return calls


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("name", list(CONFIGS))
def test_decode_steps_behind_shared_prefixes(name, graphs, shared_calls):
    config, page = CONFIGS[name]
    tiny = TinyEngine(config, page, torch.bfloat16, "cuda:0", num_pages=120, max_requests=9)
    tiny.runner.use_graphs = graphs
    cache, runner = tiny.cache, tiny.runner
    prefixes = {"p": random_prompt(config.vocab_size, 5 * page, 1), "q": random_prompt(config.vocab_size, 3 * page, 2)}
    for prefix, tokens in prefixes.items():
        cache.create_request(prefix)
        runner.step([StepEntry(prefix, tokens)])
    texts = {}
    for i, source in enumerate("ppqpq-"):
        texts[f"r{i}"] = list(prefixes.get(source, [])) + random_prompt(config.vocab_size, 1 + 7 * i, 10 + i)
        cache.create_request(f"r{i}", prefix=(source, len(prefixes[source])) if source != "-" else None)
        held = cache.get(f"r{i}").committed
        runner.step([StepEntry(f"r{i}", texts[f"r{i}"][held:])])
    # the same sizes of groups with other members, then other sizes
    batches = [("r0", "r1", "r2", "r4", "r5"), ("r0", "r1", "r2", "r4", "r5"), ("r3", "r1", "r5", "r4", "r2"), ("r4", "r0", "r2", "r3", "r5"),
               ("r0", "r1", "r3", "r5"), ("r0", "r2", "r5"), ("r1", "r0", "r3", "r2", "r4", "r5"), ("r0", "r1", "r2", "r4", "r5")]
    for turn, batch in enumerate(batches):
        for request in batch:
            texts[request].append(int(random_prompt(config.vocab_size, 1, 100 * turn + int(request[1]))[0]))
        logits = runner.step([StepEntry(request, texts[request][-1:], [0]) for request in batch])
        runner.check_device()
        for row, request in enumerate(batch):
            want = tiny.plain_logits(texts[request])[-1]
            assert_close(logits[row][None], want[None], torch.bfloat16, f"turn {turn} {request}")
    assert shared_calls and (5 * page,) in shared_calls and (5 * page, 3 * page) in shared_calls
    if graphs:
        assert runner.graph_replays >= 3
    cache.check_consistency()


def test_captured_steps_of_many_group_sizes_are_bounded(shared_calls):
    config, page = CONFIGS["E"]
    tiny = TinyEngine(config, page, torch.bfloat16, "cuda:0", num_pages=80, max_requests=9)
    tiny.runner.graph_max_shared = 2
    cache, runner = tiny.cache, tiny.runner
    prefix = random_prompt(config.vocab_size, 2 * page, 1)
    cache.create_request("p")
    runner.step([StepEntry("p", prefix)])
    texts = {f"r{i}": prefix + [i + 1] for i in range(6)}
    for name, text in texts.items():
        cache.create_request(name, prefix=("p", 2 * page))
        runner.step([StepEntry(name, text[2 * page:])])
    for turn, count in enumerate((2, 3, 4, 2, 5, 2, 3, 6, 2)):
        for _ in range(2):
            batch = list(texts)[:count]
            for name in batch:
                texts[name].append(7 * turn + 1)
            logits = runner.step([StepEntry(name, texts[name][-1:], [0]) for name in batch])
            for row, name in enumerate(batch):
                assert_close(logits[row][None], tiny.plain_logits(texts[name])[-1][None], torch.bfloat16, f"{turn} {name}")
        assert sum(len(key) > 4 for key in runner._graphs) <= 2
    assert runner.graph_replays > 0


def engine_of(tiny, page, **options):
    engine = ContinuousBatchEngine.from_model(tiny.model, block_size=page, max_running_requests=4, max_batch_tokens=64, max_model_len=384, **options)
    engine.runner.graph_capture_after = 1
    return engine


@pytest.mark.parametrize("step_ahead", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", list(CONFIGS))
def test_the_engine_with_prefixes(name, dtype, step_ahead, shared_calls):
    """The tokens of requests that share a prefix are those of requests that bring it themselves (in 32 bits, bit for bit the same
    attention; in bfloat16 up to choices closer than rounding, so the first token, which no decode step touches, and the lengths)."""
    config, page = CONFIGS[name]
    tiny = TinyEngine(config, page, dtype, "cuda:0")
    prefix = random_prompt(config.vocab_size, 4 * page + 3, 1)
    tails = [random_prompt(config.vocab_size, n, n) for n in (1, 9, 40, 3, 17)]
    rules = [dict(), dict(repetition_penalty=1.3), dict(logit_bias={7: 1.0}), dict(), dict(frequency_penalty=0.2)]
    outputs = []
    for shared in (True, False):
        engine = engine_of(tiny, page, step_ahead=step_ahead, logit_rules=True, max_prefixes=int(shared))
        if shared:
            assert engine.add_prefix("system", prefix) == 4 * page
        for i, (tail, rule) in enumerate(zip(tails, rules)):
            engine.submit(f"r{i}", prefix + tail, max_new_tokens=12, prefix="system" if shared else None, **rule)
        engine.run()
        outputs.append([list(engine.scheduler.get_request(f"r{i}").generated_token_ids) for i in range(5)])
        engine.manager.check_consistency()
        if shared:
            engine.drop_prefix("system")
        assert engine.manager.stats().free_pages == engine.manager.stats().total_pages
    assert bool(shared_calls) == (dtype == torch.bfloat16)
    if dtype == torch.float32:
        assert outputs[0] == outputs[1]
    else:
        assert [(o[0], len(o)) for o in outputs[0]] == [(o[0], len(o)) for o in outputs[1]]


@pytest.mark.parametrize("step_ahead", [False, True])
def test_a_prefix_that_comes_while_others_run(step_ahead, shared_calls):
    config, page = CONFIGS["E"]
    tiny = TinyEngine(config, page, torch.float32, "cuda:0")
    prefix = random_prompt(config.vocab_size, 3 * page, 1)
    others = [random_prompt(config.vocab_size, n, n) for n in (5, 20)]
    outputs = []
    for shared in (True, False):
        engine = engine_of(tiny, page, step_ahead=step_ahead, max_prefixes=1)
        for i, other in enumerate(others):
            engine.submit(f"o{i}", other, max_new_tokens=20)
        for _ in range(6):
            engine.step()
        if shared:
            engine.add_prefix("late", prefix)
        for i in range(2):
            engine.submit(f"s{i}", prefix + [i + 1], max_new_tokens=9, prefix="late" if shared else None)
        engine.run()
        outputs.append([list(engine.scheduler.get_request(name).generated_token_ids) for name in ("o0", "o1", "s0", "s1")])
    assert outputs[0] == outputs[1]


def test_below_the_rule_decode_steps_stay_as_they_were(monkeypatch):
    """Prefixes that save little: the fused decode attention, on shared pages."""
    config, page = CONFIGS["E"]
    tiny = TinyEngine(config, page, torch.bfloat16, "cuda:0")
    monkeypatch.setattr(ops.current(), "shared_prefix_attention", lambda *args: pytest.fail("saves too little"))
    engine = engine_of(tiny, page, max_prefixes=1)
    prefix = random_prompt(config.vocab_size, 2 * page, 1)
    engine.add_prefix("system", prefix)
    for i in range(3):
        engine.submit(f"r{i}", prefix + [i + 1], max_new_tokens=8, prefix="system")
    engine.run()
    assert engine.runner.graph_replays > 0
