"""Requests with rules on their logits through the engine and the command line on the device: captured steps, slots handed on, steps
ahead, grammars."""

from __future__ import annotations

import json
import math

import pytest
import torch

from harness import TinyEngine, random_prompt
from mini_llm_runtime_b200.engine import ContinuousBatchEngine
from mini_llm_runtime_b200.sampling import SamplingParams
from mini_llm_runtime_b200.weights import read_checkpoint
from rules_support import plain_run
from test_cli_gpu import run_cli
from test_logit_rules_engine_cpu import RULES
from tiny_configs import TINY

pytestmark = pytest.mark.gpu


def engine_of(tiny, name="A", **options):
    engine = ContinuousBatchEngine.from_model(tiny.model, block_size=TINY[name][1], max_running_requests=3, max_batch_tokens=24,
                                              max_model_len=96, logit_rules=True, **options)
    engine.runner.graph_capture_after = 1
    return engine


@pytest.mark.parametrize("step_ahead", [False, True])
@pytest.mark.parametrize("name", ["A", "B"])
def test_rules_through_the_engine(name, step_ahead):
    config, page = TINY[name]
    tiny = TinyEngine(config, page, torch.float32, "cuda:0")
    engine = engine_of(tiny, name, step_ahead=step_ahead)
    prompts = [random_prompt(config.vocab_size, n, n) for n in (5, 30, 17, 9, 33)]
    for i, (prompt, rules) in enumerate(zip(prompts, RULES)):
        engine.submit(f"r{i}", prompt, max_new_tokens=12, **rules)
    engine.run()
    assert engine.runner.graph_replays > 0
    for i, (prompt, rules) in enumerate(zip(prompts, RULES)):
        want, gap = plain_run(tiny.tensors, tiny.config_dict, SamplingParams(**rules), prompt, 12)
        assert gap > 1e-4, "the case must not hang on a rounding"
        assert list(engine.scheduler.get_request(f"r{i}").generated_token_ids) == want, (i, rules)


@pytest.mark.parametrize("temperature", [0.0, 1.3])
def test_grammars_and_bans_hold_in_bfloat16(temperature):
    config, page = TINY["A"]
    tiny = TinyEngine(config, page, torch.bfloat16, "cuda:0")
    engine = engine_of(tiny)
    prompt = random_prompt(config.vocab_size, 8, 2)
    banned = {t: -math.inf for t in range(0, config.vocab_size, 2)}
    banned = dict(list(banned.items())[:100])
    engine.submit("banned", prompt, max_new_tokens=30, temperature=temperature, logit_bias=banned)
    engine.submit("once", prompt, max_new_tokens=30, temperature=temperature, presence_penalty=1e6)
    engine.submit("bound", prompt, max_new_tokens=30, temperature=temperature)
    engine.allow_tokens("bound", [7])
    turn = 0
    while engine.scheduler.has_unfinished_requests:
        engine.step()
        output = engine.scheduler.get_request("bound").generated_token_ids
        if engine.scheduler.get_request("bound").finish_reason is None and output:
            turn += 1
            assert output[-1] == 7 if turn == 1 else output[-1] in (turn - 1, turn + 99)
            engine.allow_tokens("bound", [turn, turn + 100])
    outputs = {name: engine.scheduler.get_request(name).generated_token_ids for name in ("banned", "once", "bound")}
    assert not set(outputs["banned"]) & set(banned)
    assert len(set(outputs["once"])) == 30, "no token twice under a penalty above every logit"


def test_the_command_line(tmp_path):
    config, page = TINY["A"]
    (tmp_path / "config.json").write_text(json.dumps(config.to_dict()))
    model = tmp_path / "model"
    run_cli("make-random", "--config", str(tmp_path / "config.json"), "--seed", "12", "--out", str(model))
    prompt = [5, 17, 3, 200, 41, 9, 9, 120]
    sampling = SamplingParams(repetition_penalty=1.5, frequency_penalty=0.25, logit_bias={9: -math.inf, 33: 0.5})
    want, gap = plain_run(read_checkpoint(model), config.to_dict(), sampling, prompt, 6)
    assert gap > 1e-4
    options = ["--model", str(model), "--dtype", "float32", "--block-size", str(page), "--max-model-len", "128", "--repetition-penalty", "1.5",
               "--frequency-penalty", "0.25", "--logit-bias", "9:-inf,33:0.5", "--prompt-ids", ",".join(map(str, prompt))]
    single = json.loads(run_cli("generate", *options, "--max-new-tokens", "6").strip().splitlines()[-1])
    assert single["generated_ids"] == want
    burst = json.loads(run_cli("serve-batch", *options, "--request-count", "3", "--generation-lengths", "6").strip().splitlines()[-1])
    assert all(tokens == want for tokens in burst["runs"][0]["outputs"].values())
