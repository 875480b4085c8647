"""Requests with rules on their logits through the engine on the CPU, with stand-ins for the kernels: penalties, biases and
grammars against the plain loop, slots that are handed on, a step that fails, what is refused."""

from __future__ import annotations

import math

import pytest
import torch

from harness import TinyEngine, random_prompt
from mini_llm_runtime_b200 import ops
from mini_llm_runtime_b200.engine import ContinuousBatchEngine
from mini_llm_runtime_b200.ops import KernelError, cuda_ops
from mini_llm_runtime_b200.sampling import LogitRules, SamplingParams
from rules_support import RuledFakeOps, plain_run
from tiny_configs import TINY


@pytest.fixture(autouse=True)
def stand_in_kernels(monkeypatch):
    def need(tensor, name, dtype=None, dims=None):
        if not isinstance(tensor, torch.Tensor) or (dtype is not None and tensor.dtype != dtype) or (dims is not None and tensor.dim() != dims):
            raise KernelError(name)

    monkeypatch.setattr(cuda_ops, "_need", need)
    with ops.use(RuledFakeOps()):
        yield


def engine_of(tiny, **options):
    _, page = TINY["A"]
    return ContinuousBatchEngine.from_model(tiny.model, block_size=page, max_running_requests=2, max_batch_tokens=24, max_model_len=96,
                                            logit_rules=True, **options)


@pytest.fixture
def tiny():
    config, page = TINY["A"]
    return TinyEngine(config, page, torch.float32, "cpu")


RULES = [dict(repetition_penalty=1.8), dict(presence_penalty=0.4, frequency_penalty=0.3), dict(logit_bias={3: 2.5, 200: -math.inf, 9: 0.5}),
         dict(), dict(repetition_penalty=0.7, frequency_penalty=-0.2, logit_bias={17: 0.8})]


@pytest.mark.parametrize("step_ahead", [False, True])
def test_rules_through_the_engine(tiny, step_ahead):
    """Five requests over two slots, prompts in portions: every request's tokens are those of the plain loop with its rules."""
    config, _ = TINY["A"]
    engine = engine_of(tiny, step_ahead=step_ahead)
    prompts = [random_prompt(config.vocab_size, n, n) for n in (5, 30, 17, 9, 33)]
    for i, (prompt, rules) in enumerate(zip(prompts, RULES)):
        engine.submit(f"r{i}", prompt, max_new_tokens=6, **rules)
    engine.run()
    for i, (prompt, rules) in enumerate(zip(prompts, RULES)):
        want, gap = plain_run(tiny.tensors, tiny.config_dict, SamplingParams(**rules), prompt, 6)
        assert gap > 1e-4, "the case must not hang on a rounding"
        assert list(engine.scheduler.get_request(f"r{i}").generated_token_ids) == want, (i, rules)


def test_a_grammar_that_follows_the_tokens(tiny):
    """Even tokens after odd ones and the other way round, for one request, beside a free one; named before it is admitted and
    after each token."""
    config, _ = TINY["A"]
    engine = engine_of(tiny)
    prompt = random_prompt(config.vocab_size, 8, 2)

    def allowed_after(output):
        parity = 0 if not output else 1 - output[-1] % 2
        return set(range(parity, config.vocab_size, 2))

    engine.submit("free", prompt, max_new_tokens=7)
    engine.submit("bound", prompt, max_new_tokens=5)
    engine.allow_tokens("bound", allowed_after([]))
    while engine.scheduler.has_unfinished_requests:
        engine.step()
        request = engine.scheduler.get_request("bound")
        if request.finish_reason is None:
            engine.allow_tokens("bound", allowed_after(list(request.generated_token_ids)))
    for name, count, grammar in (("free", 7, None), ("bound", 5, allowed_after)):
        want, gap = plain_run(tiny.tensors, tiny.config_dict, SamplingParams(), prompt, count, grammar)
        assert gap > 1e-4
        assert list(engine.scheduler.get_request(name).generated_token_ids) == want
    with pytest.raises(ValueError, match="finished"):
        engine.allow_tokens("bound", None)
    assert not engine._allowed


def test_a_slot_handed_on_starts_anew(tiny):
    config, _ = TINY["A"]
    engine = engine_of(tiny)
    prompt = random_prompt(config.vocab_size, 6, 5)
    engine.submit("first", prompt, max_new_tokens=3, repetition_penalty=2.0, logit_bias={1: 4.0})
    engine.submit("beside", prompt, max_new_tokens=3)
    engine.run()
    for i in range(3):
        engine.submit(f"next{i}", prompt, max_new_tokens=3)
    engine.run()
    want, _ = plain_run(tiny.tensors, tiny.config_dict, SamplingParams(), prompt, 3)
    for name in ("beside", "next0", "next1", "next2"):
        assert list(engine.scheduler.get_request(name).generated_token_ids) == want


def test_a_step_that_fails_leaves_the_rules_to_its_repetition(tiny, monkeypatch):
    config, _ = TINY["A"]
    engine = engine_of(tiny)
    prompt = random_prompt(config.vocab_size, 6, 7)
    allowed = set(range(0, config.vocab_size, 3))
    engine.submit("a", prompt, max_new_tokens=4, frequency_penalty=0.5)
    engine.allow_tokens("a", allowed)
    forward, failures = engine.runner.model.forward, [1]

    def once(ctx):
        if failures:
            failures.pop()
            raise RuntimeError("made by the test")
        return forward(ctx)

    monkeypatch.setattr(engine.runner.model, "forward", once)
    with pytest.raises(RuntimeError, match="made by the test"):
        engine.step()
    engine.run()
    want, gap = plain_run(tiny.tensors, tiny.config_dict, SamplingParams(frequency_penalty=0.5), prompt, 4, lambda output: allowed)
    assert gap > 1e-4 and list(engine.scheduler.get_request("a").generated_token_ids) == want


def test_without_rules_nothing_is_asked_of_their_kernels(tiny):
    config, page = TINY["A"]
    engine = ContinuousBatchEngine.from_model(tiny.model, block_size=page, max_running_requests=2, max_model_len=96)
    assert engine.runner.rules is None
    for call in (lambda: engine.submit("a", [1, 2], max_new_tokens=2, presence_penalty=0.1), lambda: engine.allow_tokens("a", [1])):
        with pytest.raises(ValueError, match="logit_rules=True"):
            call()
    engine.submit("b", [1, 2], max_new_tokens=2)
    engine.run()


def test_grammars_and_stepping_ahead_exclude_each_other(tiny):
    engine = engine_of(tiny, step_ahead=True)
    engine.submit("a", [1, 2], max_new_tokens=2)
    with pytest.raises(ValueError, match="steps ahead"):
        engine.allow_tokens("a", [1])


@pytest.mark.parametrize("bad", [
    dict(repetition_penalty=0.0), dict(repetition_penalty=-1), dict(repetition_penalty=math.nan), dict(presence_penalty=math.inf),
    dict(frequency_penalty="1"), dict(presence_penalty=True), dict(logit_bias={-1: 1.0}), dict(logit_bias={1.5: 1.0}),
    dict(logit_bias={1: math.nan}), dict(logit_bias={1: math.inf}), dict(logit_bias=((1, 1.0), (1, 2.0))), dict(logit_bias={256: 1.0}),
    dict(logit_bias={t: 1.0 for t in range(301)}), dict(no_such_rule=1),
    dict(repetition_penalty=1e-39), dict(repetition_penalty=1e39), dict(presence_penalty=-1e39), dict(logit_bias={1: 1e39}),      # not in 32 bits
])
def test_rules_that_are_refused(tiny, bad):
    config, _ = TINY["A"]
    assert config.vocab_size == 256 or "logit_bias" not in bad
    engine = engine_of(tiny)
    with pytest.raises((ValueError, TypeError)):
        engine.submit("a", [1, 2], max_new_tokens=2, **bad)
    assert not engine.scheduler.has_unfinished_requests


def test_words_of_allowed_tokens():
    rules = LogitRules(2, 70, "cpu")
    words = rules.words_of([0, 31, 32, 69])
    assert words.tolist() == [1 - (1 << 31), 1, 32]
    assert rules.words_of(None).tolist() == [-1, -1, -1] and rules.words_of([]).tolist() == [0, 0, 0]
    for bad in ([70], [-1]):
        with pytest.raises(ValueError):
            rules.words_of(bad)
    for bad in ((0, 70), (2, 0)):
        with pytest.raises(ValueError):
            LogitRules(*bad, "cpu")


def test_defaults_are_no_rules():
    assert not SamplingParams().has_rules and not SamplingParams(0.7, 3).has_rules
    assert SamplingParams(logit_bias={1: 0.5}).logit_bias == ((1, 0.5),) and SamplingParams(presence_penalty=-0.1).has_rules
