"""A cache in 8 bits, forked requests, moved pages and limits on what is drawn through the engine and the command line on the device: captured
and eager steps, prompts in portions, several answers to a prompt, pools that change their size."""

from __future__ import annotations

import dataclasses
import json

import pytest
import torch

from harness import TinyEngine, random_prompt
from limits_support import kept_of
from mini_llm_runtime_b200 import ops
from mini_llm_runtime_b200.cache import CacheManager
from mini_llm_runtime_b200.engine import ContinuousBatchEngine, ModelRunner, StepEntry
from test_cli_gpu import run_cli
from tiny_configs import TINY

pytestmark = pytest.mark.gpu

DEVICE = "cuda:0"


def runner_of(tiny, page, block, dtype, pages=80, requests=6):
    cache = CacheManager(tiny.model.cache_needs(), page_size=page, num_pages=pages, max_requests=requests, max_tokens_per_request=512, dtype=dtype,
                         device=DEVICE, max_step_tokens=512, quantized_block=block)
    runner = ModelRunner(tiny.model, cache)
    runner.graph_capture_after = 1
    return runner


def near(got, want, dtype, what):
    """A code is off by half a step s = amax / 127 at most, s / sqrt(12) = amax / 440 in the mean square.  The largest of a block of 16 to
    1,024 values is 2 to 4 times their mean square root, so keys and values are off by 0.9 % at most.  Two to four layers, each with an error
    through its keys and one through its values that add up like independent ones: 0.9 % * sqrt(8) = 2.6 %; rows over few keys
    average little, so twice that, 6 %.  bfloat16's own roundings make 2 % (harness.py) of it more."""
    got, want = got.float().cpu(), want.float().cpu()
    share = 0.06 if dtype == torch.float32 else 0.08
    off = (got - want).norm(dim=-1) / want.norm(dim=-1)
    assert float(off.max()) < share, f"{what}: {float(off.max()):.4f}"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name,block", [("A", 1), ("B", 8), ("D", 16), ("D", 1), ("E", 4), ("C", 16)])
def test_logits_over_a_cache_in_8_bits(name, block, dtype):
    """Prompts in portions beside decoded tokens, eager and captured; with a scale for each token the portions do not show."""
    config, page = TINY[name]
    tiny = TinyEngine(config, page, dtype, DEVICE)
    runner = runner_of(tiny, page, block, dtype)
    texts = {f"r{i}": random_prompt(config.vocab_size, n, 40 + i) for i, n in enumerate((150, 33, 70))}
    for name_, text in texts.items():
        runner.cache.create_request(name_)
    runner.step([StepEntry("r0", texts["r0"][:100])])
    logits = runner.step([StepEntry("r0", texts["r0"][100:], [49]), StepEntry("r1", texts["r1"], [32]), StepEntry("r2", texts["r2"], [69])])
    runner.check_device()
    for row, text in enumerate(texts.values()):
        near(logits[row][None], tiny.plain_logits(text)[-1][None], dtype, f"prompt {row}")
    for turn in range(5):
        for i, text in enumerate(texts.values()):
            text.append(int(random_prompt(config.vocab_size, 1, 10 * turn + i)[0]))
        logits = runner.step([StepEntry(name_, text[-1:], [0]) for name_, text in texts.items()])
        runner.check_device()
        for row, text in enumerate(texts.values()):
            near(logits[row][None], tiny.plain_logits(text)[-1][None], dtype, f"turn {turn} row {row}")
    assert runner.graph_replays >= 3
    # the same texts token by token and at once
    if dtype == torch.float32 and block == 1:
        whole = runner_of(tiny, page, block, dtype)
        for name_, text in texts.items():
            whole.cache.create_request(name_)
            mine = whole.step([StepEntry(name_, text, [len(text) - 1])])
            row = list(texts).index(name_)
            assert float((mine[0] - logits[row]).abs().max()) < 2e-3 * float(logits[row].abs().max())


def engine_of(tiny, page, **options):
    options = {"total_blocks": 60, "max_running_requests": 6, "max_batch_tokens": 64, "max_model_len": 160, **options}
    engine = ContinuousBatchEngine.from_model(tiny.model, block_size=page, **options)
    engine.runner.graph_capture_after = 1
    return engine


@pytest.mark.parametrize("cache", [{}, {"cache_dtype": "int8"}, {"cache_dtype": "int8", "cache_block": 8}])
@pytest.mark.parametrize("step_ahead", [False, True])
def test_several_limited_answers_out_of_one_cache(cache, step_ahead):
    """Several answers to each prompt, drawn under limits, out of pages held together, while the pools change their size: each as if it had the
    engine to itself."""
    config, page = TINY["A"]
    tiny = TinyEngine(config, page, torch.float32, DEVICE)
    prompts = [random_prompt(config.vocab_size, n, n) for n in (45, 6)]
    limits = {"temperature": 1.3, "top_k": 30, "top_p": 0.9, "min_p": 0.01}
    engine = engine_of(tiny, page, sampling_limits=True, step_ahead=step_ahead, **cache)
    got = engine.generate(prompts, max_new_tokens=8, seed=11, answers=3, **limits)
    engine.runner.check_device()
    assert engine.runner.graph_replays > 0
    assert engine.manager.stats().free_pages == (60,) and engine.manager.stats().promised_pages == (0,)
    want = []
    alone = engine_of(tiny, page, sampling_limits=True, **cache)
    for i, prompt in enumerate(prompts):
        for j in range(3):
            want += alone.generate([prompt], max_new_tokens=8, seed=11 + 3 * i + j, **limits)
    if cache.get("cache_block", 1) == 1:
        assert got == want
    assert len({tuple(answer) for answer in got}) > 3


@pytest.mark.parametrize("step_ahead", [False, True])
def test_pools_that_change_their_size_while_requests_run(step_ahead):
    config, page = TINY["A"]
    tiny = TinyEngine(config, page, torch.float32, DEVICE)
    prompts = {name: random_prompt(config.vocab_size, n, n) for name, n in (("a", 40), ("b", 17), ("c", 60))}
    for cache in ({}, {"cache_dtype": "int8", "cache_block": 16}):
        still, moved = (engine_of(tiny, page, step_ahead=step_ahead, **cache) for _ in range(2))
        for engine in (still, moved):
            for name, prompt in prompts.items():
                engine.submit(name, prompt, max_new_tokens=12)
            for turn in range(12):
                if engine is moved and turn in (2, 5, 7):
                    engine.resize_cache({2: 14, 5: 100, 7: 13}[turn])
                    engine.manager.compact()
                    engine.manager.check_consistency()
                engine.step()
            engine.run()
            engine.runner.check_device()
        for name in prompts:
            assert moved.scheduler.get_request(name).generated_token_ids == still.scheduler.get_request(name).generated_token_ids


@pytest.mark.parametrize("name", ["A", "D"])
def test_every_token_lies_within_the_limits(name):
    """In bfloat16, captured: every drawn token is one of those that the limits leave of its step's logits (or beside a border that the logits' own
    rounding could move: none of these cases is)."""
    config, page = TINY[name]
    config = dataclasses.replace(config, use_sliding_window=False)
    tiny = TinyEngine(config, page, torch.bfloat16, DEVICE)
    engine = engine_of(tiny, page, sampling_limits=True)
    limits = [{"top_k": 3}, {"top_p": 0.3}, {"min_p": 0.5}, {"top_k": 40, "top_p": 0.8}, {}]
    for i, own in enumerate(limits):
        engine.submit(f"r{i}", random_prompt(config.vocab_size, 5 + i, i), max_new_tokens=10, temperature=0.8, seed=i, **own)
    seen = 0
    step = engine.runner.step

    def watched(entries, **options):
        logits, tokens = step(entries, **options)
        rows = [e.request_id for e in entries if len(e.want)]
        for row, request in enumerate(rows):
            own = limits[int(request[1:])]
            kept, _, _ = kept_of(logits[row], float(torch.tensor(0.8)), own.get("top_k", 0), float(torch.tensor(own.get("top_p", 1.0))),
                                 float(torch.tensor(own.get("min_p", 0.0))))
            assert int(tokens[row]) in kept.tolist(), (request, own)
            nonlocal seen
            seen += 1
        return logits, tokens

    engine.runner.step = watched
    engine.run()
    assert seen == 50 and engine.runner.graph_replays > 0


def test_limits_on_the_command_line(tmp_path):
    config, _ = TINY["A"]
    (tmp_path / "config.json").write_text(json.dumps(config.to_dict()))
    model = tmp_path / "model"
    run_cli("make-random", "--config", str(tmp_path / "config.json"), "--out", str(model))
    outputs = []
    for options in ((), ("--temperature", "3", "--top-k", "1"), ("--temperature", "3", "--top-p", "0.000001"), ("--temperature", "3", "--seed", "4")):
        done = run_cli("generate", "--model", str(model), "--dtype", "float32", "--max-model-len", "128", "--prompt-ids", "3,1,4,1,5", "--max-new-tokens", "6", *options)
        outputs.append(json.loads(done.splitlines()[-1])["generated_ids"])
    assert outputs[0] == outputs[1] == outputs[2] != outputs[3]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("page,block,heads,kv_heads,dim", [(16, 1, 6, 2, 64), (8, 4, 3, 3, 20), (32, 16, 8, 1, 128)])
def test_turned_and_stored_in_8_bits_as_in_two_calls(page, block, heads, kv_heads, dim, dtype):
    kernels = ops.current()
    generator = torch.Generator(device=DEVICE).manual_seed(5)
    # blocks in any order, the rows of each one behind the other, the first one's from its middle on, the last one's not to its end
    blocks = torch.randperm(6 * page // block, generator=generator, device=DEVICE)[:max(3, 37 // block)]
    slots = (blocks[:, None] * block + torch.arange(block, device=DEVICE)).reshape(-1)[block // 2:][:-(block // 3) or None].contiguous()
    rows = len(slots)
    qkv = torch.randn(rows, (heads + 2 * kv_heads) * dim, generator=generator, device=DEVICE).to(dtype)
    positions = torch.randint(0, 400, (rows,), generator=generator, device=DEVICE, dtype=torch.int32)
    frequencies = 10000.0 ** (-torch.arange(dim // 2, device=DEVICE, dtype=torch.float32) / (dim // 2))

    def pool():
        codes = [torch.zeros(6, kv_heads, page, dim, dtype=torch.int8, device=DEVICE) for _ in range(2)]
        scales = [torch.zeros(6, kv_heads, page // block, device=DEVICE) for _ in range(2)]
        return ops.QuantizedPool(*codes, *scales)

    one, two = pool(), pool()
    q = kernels.rope_quantize_kv_write(qkv, positions, frequencies, slots, one, heads, kv_heads, dim)
    # one page of `rows` tokens holds the turned keys and the values, head by head
    turned = [torch.zeros(1, kv_heads, rows, dim, dtype=dtype, device=DEVICE) for _ in range(2)]
    want = kernels.rope_kv_write(qkv, positions, frequencies, torch.arange(rows, device=DEVICE), *turned, heads, kv_heads, dim)
    kernels.quantize_kv_write(*(t[0].transpose(0, 1).reshape(rows, kv_heads * dim).contiguous() for t in turned), slots, two)
    assert torch.equal(q, want)
    for a, b in zip((one.key, one.value, one.key_scales, one.value_scales), (two.key, two.value, two.key_scales, two.value_scales)):
        assert torch.equal(a, b)
    untouched = pool()
    again = kernels.rope_quantize_kv_write(qkv, positions, frequencies, slots, untouched, heads, kv_heads, dim, write_kv=False)
    assert torch.equal(again, want) and not untouched.key.any() and not untouched.value_scales.any()
    kernels.raise_if_device_error()


def test_refusals_of_what_turns_and_stores():
    kernels = ops.current()
    pool = ops.QuantizedPool(*(torch.zeros(2, 2, 8, 16, dtype=torch.int8, device=DEVICE) for _ in range(2)),
                             *(torch.zeros(2, 2, 8, device=DEVICE) for _ in range(2)))
    qkv = torch.zeros(3, 8 * 16, device=DEVICE)
    positions, slots = torch.zeros(3, dtype=torch.int32, device=DEVICE), torch.arange(3, device=DEVICE)
    frequencies = torch.ones(8, device=DEVICE)
    call = lambda **other: kernels.rope_quantize_kv_write(**{**dict(qkv=qkv, positions=positions, inv_freq=frequencies, slots=slots, pool=pool,
                                                                    num_heads=4, num_kv_heads=2, head_dim=16), **other})
    call()
    for other in ({"num_heads": 3}, {"head_dim": 32}, {"positions": positions[:2]}, {"slots": slots[:2]}, {"slots": slots.int()},
                  {"inv_freq": frequencies[:4]}, {"num_kv_heads": 1, "num_heads": 6}, {"qkv": qkv.half()}, {"qkv": qkv.cpu()}, {"qkv": qkv[None]}):
        with pytest.raises((ops.KernelError, ValueError, TypeError)):
            call(**other)
    assert call(qkv=qkv[:0], positions=positions[:0], slots=slots[:0]).shape == (0, 64)


@pytest.mark.parametrize("cache", [{}, {"cache_dtype": "int8"}])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_all_of_it_in_one_engine(cache, dtype):
    """A shared prefix, a fork of a request that starts with it, a fork of one that has ended, rules and limits beside one another: in float32 each
    request's tokens are those it gets alone, in bfloat16 all run to their ends."""
    config, page = TINY["D"]
    config = dataclasses.replace(config, use_sliding_window=False)
    tiny = TinyEngine(config, page, dtype, DEVICE)
    options = {"sampling_limits": True, "logit_rules": True, "max_prefixes": 1, **cache}
    system = random_prompt(config.vocab_size, 40, 1)
    drawn = {"temperature": 1.1, "top_k": 25, "top_p": 0.95, "repetition_penalty": 1.2, "logit_bias": {3: -5.0, 5: float("-inf")}}
    prompts = {"a": system + [7, 8, 9], "b": system + [7, 8, 9], "c": system[:21] + [1, 2], "d": random_prompt(config.vocab_size, 9, 2)}
    engine = engine_of(tiny, page, **options)
    assert engine.add_prefix("system", system) == 32
    engine.submit("d", prompts["d"], max_new_tokens=2, seed=4)
    engine.submit("a", prompts["a"], max_new_tokens=14, seed=1, prefix="system", **drawn)
    engine.step()
    engine.step()
    engine.submit("b", prompts["b"], max_new_tokens=14, seed=2, fork_of="a", **drawn)
    engine.submit("c", prompts["c"], max_new_tokens=14, seed=3, fork_of="a", min_p=0.1, temperature=0.9)
    engine.step()
    engine.manager.check_consistency()
    engine.run()
    engine.runner.check_device()
    engine.submit("late", prompts["d"] + list(engine.scheduler.get_request("d").generated_token_ids), max_new_tokens=5, seed=5, fork_of="d")
    engine.run()
    engine.drop_prefix("system")
    engine.manager.check_consistency()
    assert engine.manager.stats().free_pages == (60,)
    for name, how in (("a", {"seed": 1, **drawn}), ("b", {"seed": 2, **drawn}), ("c", {"seed": 3, "min_p": 0.1, "temperature": 0.9})):
        got = list(engine.scheduler.get_request(name).generated_token_ids)
        assert len(got) == 14 and (name == "c" or 5 not in got)
        if dtype == torch.float32:
            alone = engine_of(tiny, page, **options)
            assert got == alone.generate([prompts[name]], max_new_tokens=14, **how)[0], name
