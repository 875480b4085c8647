"""Forked requests, moved pages, limits on what is drawn and a cache in 8 bits on the CPU: the cache manager under random orders, and the
engine with stand-ins for the kernels."""

from __future__ import annotations

import random

import pytest
import torch

import plain_qwen2 as plain
from harness import TinyEngine, random_prompt
from mini_llm_runtime_b200 import ops
from mini_llm_runtime_b200.cache import OutOfPages
from mini_llm_runtime_b200.engine import ContinuousBatchEngine
from mini_llm_runtime_b200.ops import cuda_ops
from mini_llm_runtime_b200.sampling import SamplingParams
from requests_support import RequestFakeOps
from mini_llm_runtime_b200.cache import CacheManager
from mini_llm_runtime_b200.engine import StepEntry
from mini_llm_runtime_b200.parts import KVCacheNeed
from test_cache_manager import FULL, WINDOW
from tiny_configs import TINY

SMALL = KVCacheNeed(1, 8, None)


@pytest.fixture(autouse=True)
def kernels(monkeypatch):
    monkeypatch.setattr(cuda_ops, "_need", lambda *args, **kwargs: None)
    with ops.use(RequestFakeOps()) as stand_in:
        yield stand_in


# ------------------------------------------------------------------ the cache manager
def manager(pages, page, needs=(FULL, SMALL, FULL), requests=6):
    return CacheManager(list(needs), page_size=page, num_pages=pages, max_requests=requests, max_tokens_per_request=64, dtype=torch.float32,
                        device="cpu", max_step_tokens=16)


def write(m, request, tokens):
    """``tokens`` more of a request, their places in the pools filled with them."""
    first = m.get(request).committed
    m.begin_step([(request, len(tokens))])
    for group in m.groups:
        for i, place in enumerate(m.slot_mapping(group, m.get(request), first, len(tokens))):
            page, offset = divmod(int(place), m.page_size)
            for pool in (group.key, group.value):
                pool[:, page, :, offset] = float(tokens[i])
    m.commit_step()


def held(m, request):
    """The texts that the pools hold for a request, by group."""
    r = m.get(request)
    out = []
    for group in m.groups:
        places = m.slot_mapping(group, r, 0, r.committed)
        out.append([int(group.key[0, int(p) // m.page_size, 0, int(p) % m.page_size, 0]) for p in places])
    return out


@pytest.mark.parametrize("tokens", [1, 3, 4, 7, 8, 10])
def test_a_fork_holds_whole_pages_with_its_parent_and_copies_the_last(tokens, kernels):
    m = manager(pages=12, page=4)
    m.create_request("a")
    write(m, "a", list(range(1, 11)))
    before = m.stats().free_pages
    fork = m.create_request("b", fork=("a", tokens))
    assert fork.committed == tokens and held(m, "b") == [list(range(1, tokens + 1))] * len(m.groups)
    assert before[0] - m.stats().free_pages[0] == (1 if tokens % 4 else 0)
    assert len(kernels.copied) == (len(m.groups) if tokens % 4 else 0)
    m.check_consistency()
    write(m, "b", [50, 51, 52])
    write(m, "a", [11, 12, 13])
    assert held(m, "a")[0] == list(range(1, 14)) and held(m, "b")[0] == list(range(1, tokens + 1)) + [50, 51, 52]
    m.check_consistency()
    m.release("a")
    m.check_consistency()
    assert held(m, "b")[0] == list(range(1, tokens + 1)) + [50, 51, 52]
    m.release("b")
    assert m.stats().free_pages == tuple(g.num_pages for g in m.groups)


def test_promises_follow_the_pages():
    """A parent that ends leaves the pages that its forks hold to them, with their share of the promise."""
    m = manager(pages=10, page=4)
    m.create_request("a", lifetime_tokens=16)
    write(m, "a", list(range(1, 11)))
    assert m.create_request("b", lifetime_tokens=16, fork=("a", 10)).promised[0] == 2      # two of four pages are the parent's
    assert m.create_request("c", lifetime_tokens=12, fork=("b", 9)).promised[0] == 1
    assert m.stats().promised_pages[0] == 7
    assert m.create_request("d", lifetime_tokens=16) is None                               # four more do not fit
    m.release("a")                                                                         # its third page, and the promise of the fourth
    m.check_consistency()
    assert m.stats().promised_pages[0] == 5 and m.get("b").promised[0] == 4 and m.get("c").promised[0] == 1
    write(m, "b", list(range(60, 66)))
    write(m, "c", [70, 71, 72])
    assert held(m, "b")[0] == list(range(1, 11)) + list(range(60, 66)) and held(m, "c")[0] == list(range(1, 10)) + [70, 71, 72]
    m.release("b")
    m.check_consistency()
    assert m.get("c").promised[0] == 3 and m.stats().promised_pages[0] == 3
    m.release("c")
    assert m.stats().promised_pages[0] == 0 and m.stats().free_pages[0] == 10


def test_a_promised_request_and_an_unpromised_one_hand_pages_to_one_another():
    for first, second in (({"lifetime_tokens": 16}, {}), ({}, {"lifetime_tokens": 16})):
        m = manager(pages=9, page=4)
        m.create_request("a", **first)
        write(m, "a", list(range(1, 9)))
        m.create_request("b", fork=("a", 8), **second)
        m.release("a")
        m.check_consistency()
        write(m, "b", list(range(9, 17)))
        m.check_consistency()
        assert held(m, "b")[0] == list(range(1, 17))
        m.release("b")
        assert m.stats().promised_pages[0] == 0 and m.stats().free_pages[0] == 9


def test_a_fork_of_a_request_that_starts_with_a_prefix():
    m = manager(pages=16, page=4)
    m.create_request("p", lifetime_tokens=8, lasting=True)
    write(m, "p", list(range(1, 9)))
    m.create_request("a", lifetime_tokens=20, prefix=("p", 8))
    write(m, "a", list(range(9, 15)))
    m.create_request("b", lifetime_tokens=20, fork=("a", 13))
    m.create_request("c", lifetime_tokens=20, fork=("a", 6))
    assert m.get("p").sharers == 3 and m.get("b").shared_pages == 2 and m.get("c").shared_pages == 1
    m.check_consistency()
    m.release("a")
    m.check_consistency()
    assert held(m, "b")[0] == list(range(1, 14)) and held(m, "c")[0] == list(range(1, 7))
    for request in ("b", "c", "p"):
        m.release(request)
    assert m.stats().free_pages[0] == 16


def test_what_a_fork_refuses_leaves_everything_as_it_was():
    m = manager(pages=4, page=4, needs=[FULL])
    m.create_request("a")
    write(m, "a", list(range(1, 15)))
    before = m.stats()
    for fork, options in ((("a", 0), {}), (("a", 15), {}), (("a", 10), {"lifetime_tokens": 10}), (("a", 4), {"lasting": True, "lifetime_tokens": 9}),
                          (("a", 4), {"prefix": ("a", 4)})):
        with pytest.raises(ValueError):
            m.create_request("b", fork=fork, **options)
    with pytest.raises(KeyError):
        m.create_request("b", fork=("z", 4))
    with pytest.raises(OutOfPages):
        m.create_request("b", fork=("a", 14))            # no page for the copy
    assert m.create_request("b", fork=("a", 13), lifetime_tokens=16) is None
    assert m.stats() == before
    m.check_consistency()
    windowed = manager(pages=8, page=4, needs=[FULL, WINDOW])
    windowed.create_request("a")
    windowed.begin_step([("a", 6)])
    windowed.commit_step()
    with pytest.raises(ValueError, match="fork"):
        windowed.create_request("b", fork=("a", 5))


@pytest.mark.parametrize("seed", range(6))
def test_random_orders_of_forks_steps_releases_and_moves(seed):
    rng = random.Random(seed)
    m = manager(pages=40, page=4, requests=9)
    texts, counter = {}, 0
    for _ in range(250):
        action = rng.random()
        if action < 0.3 and len(texts) < 9:
            name, parent = f"r{counter}", rng.choice(list(texts)) if texts and rng.random() < 0.7 else None
            counter += 1
            options = {"lifetime_tokens": 40} if rng.random() < 0.5 and m.can_ever_hold(40) else {}
            try:
                if parent is None or not texts[parent]:
                    made, start = m.create_request(name, **options), []
                else:
                    tokens = rng.randrange(1, len(texts[parent]) + 1)
                    if options and tokens >= 40:
                        continue
                    made, start = m.create_request(name, fork=(parent, tokens), **options), texts[parent][:tokens]
            except OutOfPages:
                made = None
            if made is not None:
                texts[name] = list(start)
        elif action < 0.7 and texts:
            name = rng.choice(list(texts))
            count = min(rng.randrange(1, 7), 40 - len(texts[name]))
            if count > 0:
                new = [rng.randrange(1, 1000) for _ in range(count)]
                try:
                    write(m, name, new)
                    texts[name] += new
                except OutOfPages:
                    pass
        elif action < 0.85 and texts:
            name = rng.choice(list(texts))
            m.release(name)
            del texts[name]
        elif action < 0.93:
            m.compact()
            assert all(max(g.allocator.held, default=-1) < max(1, g.allocator.held_count) for g in m.groups)
        else:
            count = max(g.allocator.needed for g in m.groups) + rng.randrange(0, 12)
            m.resize(max(1, count))
            assert all(g.num_pages == max(1, count) for g in m.groups)
        m.check_consistency()
        for name, text in texts.items():
            assert held(m, name) == [text] * len(m.groups)
    for name in list(texts):
        m.release(name)
    assert all(g.allocator.free_count == g.num_pages and g.allocator.promised == 0 for g in m.groups)


def test_pools_do_not_shrink_below_what_is_promised():
    m = manager(pages=10, page=4)
    m.create_request("a", lifetime_tokens=16)
    write(m, "a", [1, 2, 3, 4, 5])
    for count in (0, 3):
        with pytest.raises(OutOfPages):
            m.resize(count)
    m.resize(4)
    write(m, "a", list(range(6, 17)))
    assert held(m, "a")[0] == list(range(1, 17))
    m.check_consistency()


# ------------------------------------------------------------------ the engine
@pytest.fixture
def tiny():
    return TinyEngine(*TINY["A"], torch.float32, "cpu")


def engine_of(tiny, **options):
    options = {"total_blocks": 40, "max_running_requests": 4, "max_batch_tokens": 64, "max_model_len": 160, **options}
    return ContinuousBatchEngine.from_model(tiny.model, block_size=TINY["A"][1], **options)


def rows_run(engine, monkeypatch):
    """How many rows each step brings to the model."""
    rows, step = [], engine.runner.step
    monkeypatch.setattr(engine.runner, "step", lambda entries, **kw: rows.append(sum(len(e.tokens) for e in entries)) or step(entries, **kw))
    return rows


def test_a_forked_request_runs_the_tokens_that_it_does_not_share(tiny, monkeypatch):
    engine = engine_of(tiny)
    rows = rows_run(engine, monkeypatch)
    prompt = random_prompt(tiny.config.vocab_size, 40, 1)
    engine.submit("a", prompt, max_new_tokens=8)
    for _ in range(3):
        engine.step()
    longer = prompt + list(engine.scheduler.get_request("a").generated_token_ids) + [5, 6]
    engine.submit("same", prompt, max_new_tokens=4, fork_of="a")
    engine.submit("longer", longer, max_new_tokens=4, fork_of="a")
    other = prompt[:20] + [prompt[20] ^ 1] + prompt[21:]
    engine.submit("other", other, max_new_tokens=4, fork_of="a")
    del rows[:]
    engine.step()
    # one decoded token; the last token of the prompt; two new ones and the last one that is not in the cache yet; 20 of the other's 40
    assert rows == [1 + 1 + 3 + 20]
    engine.manager.check_consistency()
    engine.run()
    for name, text, count in (("a", prompt, 8), ("same", prompt, 4), ("longer", longer, 4), ("other", other, 4)):
        assert list(engine.scheduler.get_request(name).generated_token_ids) == plain.greedy_tokens(tiny.tensors, tiny.config_dict, text, count), name
    assert engine.manager.stats().free_pages == (40,) and engine.manager.stats().promised_pages == (0,)


def test_a_fork_of_a_request_that_has_ended_is_computed(tiny, monkeypatch):
    engine = engine_of(tiny)
    prompt = random_prompt(tiny.config.vocab_size, 30, 2)
    engine.submit("a", prompt, max_new_tokens=2)
    engine.run()
    rows = rows_run(engine, monkeypatch)
    engine.submit("b", prompt, max_new_tokens=2, fork_of="a")
    engine.run()
    assert rows[0] == 30
    assert engine.scheduler.get_request("b").generated_token_ids == engine.scheduler.get_request("a").generated_token_ids


def test_a_failed_step_gives_a_fork_back_and_it_starts_again(tiny, monkeypatch):
    engine = engine_of(tiny)
    prompt = random_prompt(tiny.config.vocab_size, 30, 3)
    engine.submit("a", prompt, max_new_tokens=6)
    engine.step()
    engine.submit("b", prompt, max_new_tokens=3, fork_of="a")
    forward = engine.runner.model.forward
    monkeypatch.setattr(engine.runner.model, "forward", lambda ctx: (_ for _ in ()).throw(RuntimeError("fails")))
    with pytest.raises(RuntimeError, match="fails"):
        engine.step()
    engine.manager.check_consistency()
    monkeypatch.setattr(engine.runner.model, "forward", forward)
    engine.run()
    for name, count in (("a", 6), ("b", 3)):
        assert list(engine.scheduler.get_request(name).generated_token_ids) == plain.greedy_tokens(tiny.tensors, tiny.config_dict, prompt, count)


@pytest.mark.parametrize("config", ["A", "C"])
def test_several_answers_are_those_of_requests_by_themselves(config, monkeypatch):
    """Model C has windows: its answers are computed each by itself."""
    tiny = TinyEngine(*TINY[config], torch.float32, "cpu")
    prompts = [random_prompt(tiny.config.vocab_size, n, n) for n in (37, 5)]
    limits = {"temperature": 1.5, "top_k": 20, "top_p": 0.9}
    engine = engine_of(tiny, sampling_limits=True, total_blocks=60, max_running_requests=6)
    rows = rows_run(engine, monkeypatch)
    got = engine.generate(prompts, max_new_tokens=5, seed=7, answers=3, **limits)
    if config == "A":
        assert sum(rows) == 42 + 4 * 1 + 6 * 4      # each prompt once, its last token for each further answer, four tokens fed back each
    want = []
    for i, prompt in enumerate(prompts):
        for j in range(3):
            alone = engine_of(tiny, sampling_limits=True)
            want += alone.generate([prompt], max_new_tokens=5, seed=7 + 3 * i + j, **limits)
    assert got == want and len({tuple(answer) for answer in got}) > 2
    assert engine.manager.stats().free_pages == (60,) * len(engine.manager.groups)


def test_limits_go_with_their_requests(tiny):
    engine = engine_of(tiny, sampling_limits=True)
    prompt = random_prompt(tiny.config.vocab_size, 9, 4)
    engine.submit("one", prompt, max_new_tokens=6, temperature=3.0, top_k=1)
    engine.submit("small", prompt, max_new_tokens=6, temperature=3.0, top_p=1e-6)
    engine.submit("sure", prompt, max_new_tokens=6, temperature=3.0, min_p=1.0)
    engine.submit("free", prompt, max_new_tokens=6, temperature=3.0, seed=5)
    engine.run()
    want = plain.greedy_tokens(tiny.tensors, tiny.config_dict, prompt, 6)
    for name in ("one", "small", "sure"):
        assert list(engine.scheduler.get_request(name).generated_token_ids) == want
    assert list(engine.scheduler.get_request("free").generated_token_ids) != want
    # the slots' next requests bring none
    engine.submit("next", prompt, max_new_tokens=6, temperature=3.0, seed=5)
    engine.run()
    assert engine.scheduler.get_request("next").generated_token_ids == engine.scheduler.get_request("free").generated_token_ids


def test_what_submit_refuses(tiny):
    engine = engine_of(tiny)
    prompt = random_prompt(tiny.config.vocab_size, 9, 4)
    engine.submit("a", prompt, max_new_tokens=2)
    with pytest.raises(ValueError, match="sampling_limits"):
        engine.submit("b", prompt, max_new_tokens=2, top_k=5)
    with pytest.raises(KeyError):
        engine.submit("b", prompt, max_new_tokens=2, fork_of="z")
    with pytest.raises(ValueError, match="itself"):
        engine.submit("b", prompt, max_new_tokens=2, fork_of="b")
    with pytest.raises(ValueError, match="exclude"):
        engine.submit("b", prompt, max_new_tokens=2, fork_of="a", prefix="p")
    with pytest.raises(ValueError, match="answers"):
        engine.generate([prompt], max_new_tokens=2, answers=0)
    with pytest.raises(ValueError, match="int8"):
        engine_of(tiny, cache_dtype="fp8")
    windowed = TinyEngine(*TINY["C"], torch.float32, "cpu")
    engine = ContinuousBatchEngine.from_model(windowed.model, block_size=16, total_blocks=20, max_running_requests=2, max_batch_tokens=32, max_model_len=96)
    engine.submit("a", [1, 2, 3], max_new_tokens=2)
    with pytest.raises(ValueError, match="fork"):
        engine.submit("b", [1, 2, 3], max_new_tokens=2, fork_of="a")
    for bad in ({"top_k": -1}, {"top_k": 1.5}, {"top_k": True}, {"top_p": 0.0}, {"top_p": 1.5}, {"top_p": float("nan")}, {"min_p": -0.1},
                {"min_p": 2.0}, {"min_p": "x"}):
        with pytest.raises(ValueError):
            SamplingParams(**bad)
    assert SamplingParams(top_k=3).has_limits and not SamplingParams(temperature=2.0).has_limits


def test_a_cache_that_changes_its_size_between_steps(tiny):
    engine = engine_of(tiny, total_blocks=20)
    prompts = {name: random_prompt(tiny.config.vocab_size, n, n) for name, n in (("a", 33), ("b", 20), ("c", 50))}
    for name in ("a", "b", "c"):
        engine.submit(name, prompts[name], max_new_tokens=7)
    for size in (20, 12, 40, 11):
        engine.step()
        engine.resize_cache(size)
        engine.manager.check_consistency()
        assert engine.manager.groups[0].num_pages == size
    with pytest.raises(OutOfPages):
        engine.resize_cache(5)
    engine.submit("d", random_prompt(tiny.config.vocab_size, 100, 1), max_new_tokens=30)
    with pytest.raises(OutOfPages, match="never be admitted|held or promised"):
        engine.resize_cache(8)
    engine.resize_cache(30)
    engine.run()
    for name, prompt in prompts.items():
        assert list(engine.scheduler.get_request(name).generated_token_ids) == plain.greedy_tokens(tiny.tensors, tiny.config_dict, prompt, 7)


@pytest.mark.parametrize("block", [1, 4, 16])
def test_a_cache_in_8_bits_keeps_the_logits_near(tiny, block):
    """Keys and values are off by half a step, 1/254 of their block's largest, of each: the first tokens' logits by little."""
    engine = engine_of(tiny, cache_dtype="int8", cache_block=block)
    assert all(group.key.dtype == torch.int8 and group.key_scales.shape[-1] == 16 // block for group in engine.manager.groups)
    exact = engine_of(tiny)
    prompt = random_prompt(tiny.config.vocab_size, 45, 8)
    logits = []
    for e in (engine, exact):
        e.manager.create_request("x")
        first = e.runner.step([StepEntry("x", prompt[:30], [29])])
        second = e.runner.step([StepEntry("x", prompt[30:], [14])])
        logits.append(torch.cat([first, second]))
    scale = float(logits[1].abs().max())
    assert 0 < float((logits[0] - logits[1]).abs().max()) < 0.05 * scale


def test_cuts_do_not_show_in_a_cache_with_a_scale_for_each_token(tiny):
    prompt = random_prompt(tiny.config.vocab_size, 40, 9)
    results = []
    for cuts in ((40,), (7, 16, 17), (1, 2, 37)):
        engine = engine_of(tiny, cache_dtype="int8")
        engine.manager.create_request("x")
        at, rows = 0, []
        for cut in (*cuts, 40):
            if cut > at:
                rows.append(engine.runner.step([StepEntry("x", prompt[at:cut], [cut - at - 1])])[0])
                at = cut
        results.append((rows[-1], [p.clone() for g in engine.manager.groups for p in g.pools]))
    for logits, pools in results[1:]:
        assert torch.allclose(logits, results[0][0], atol=2e-5 * float(results[0][0].abs().max()))
    sizes = [int((a != b).sum()) for pools in (results[1][1], results[2][1]) for a, b in zip(pools, results[0][1])]
    assert all(s <= 4 for s in sizes[0::4] + sizes[1::4])       # codes, but for a number beside a tie (32-bit sums differ by the cut)


def test_blocks_divide_pages_and_other_attention_refuses_a_cache_in_8_bits():
    with pytest.raises(ValueError, match="divide"):
        CacheManager([FULL], page_size=16, num_pages=2, max_requests=1, max_tokens_per_request=16, dtype=torch.float32, device="cpu", quantized_block=5)
    with pytest.raises(ValueError, match="one size"):
        CacheManager([KVCacheNeed(2, 16, None, value_dim=8)], page_size=16, num_pages=2, max_requests=1, max_tokens_per_request=16, dtype=torch.float32,
                     device="cpu", quantized_block=16)
    tiny = TinyEngine(*TINY["A"], torch.float32, "cpu")
    tiny.model.blocks[0].mixer.supports_quantized_cache = False
    with pytest.raises(ValueError, match="8 bits"):
        engine_of(tiny, cache_dtype="int8")
