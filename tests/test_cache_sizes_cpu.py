"""Pools that change their size: what a call that fails leaves, and which sizes an engine with waiting requests and prefixes takes."""

from __future__ import annotations

import pytest
import torch

import plain_qwen2 as plain
from harness import TinyEngine, random_prompt
from mini_llm_runtime_b200 import ops
from mini_llm_runtime_b200.cache import CacheManager, OutOfPages
from mini_llm_runtime_b200.ops import KernelError, cuda_ops
from requests_support import RequestFakeOps
from test_cache_manager import FULL
from test_forked_requests_cpu import SMALL, engine_of, held, write
from tiny_configs import TINY


@pytest.fixture(autouse=True)
def kernels(monkeypatch):
    monkeypatch.setattr(cuda_ops, "_need", lambda *args, **kwargs: None)
    with ops.use(RequestFakeOps()) as stand_in:
        yield stand_in


def filled(block):
    m = CacheManager([FULL, SMALL, FULL], page_size=4, num_pages=6, max_requests=3, max_tokens_per_request=64, dtype=torch.float32, device="cpu",
                     max_step_tokens=16, quantized_block=block)
    for name, tokens in (("a", range(1, 8)), ("b", range(20, 25)), ("c", range(30, 33))):
        m.create_request(name)
        write(m, name, list(tokens))
    m.release("b")
    return m


@pytest.mark.parametrize("block", [None, 2])
@pytest.mark.parametrize("count", [12, 3])
def test_a_resize_that_runs_out_of_memory_leaves_the_cache_as_it_was(block, count, monkeypatch):
    """Every allocation of the new pools fails once, the one after it not."""
    zeros = torch.zeros
    for failing in range((4 if block else 2) * 2):
        m = filled(block)
        before = [[(pool, pool.clone()) for pool in group.pools] for group in m.groups]
        quantized, stats = [list(group.quantized) for group in m.groups], m.stats()
        calls = [0]

        def some(*args, **kwargs):
            calls[0] += 1
            if calls[0] == failing + 1:
                raise torch.OutOfMemoryError("no room")
            return zeros(*args, **kwargs)

        monkeypatch.setattr(torch, "zeros", some)
        with pytest.raises(torch.OutOfMemoryError):
            m.resize(count)
        monkeypatch.setattr(torch, "zeros", zeros)
        for group, pools, entries in zip(m.groups, before, quantized):
            assert group.num_pages == 6 and group.allocator.total == 6 and group.quantized == entries
            assert all(now is pool and torch.equal(now, copy) for now, (pool, copy) in zip(group.pools, pools))
        assert m.stats() == stats
        m.check_consistency()
        m.resize(count)
        m.check_consistency()
        assert held(m, "a")[0] == list(range(1, 8)) and held(m, "c")[0] == [30, 31, 32]
        for group in m.groups:
            assert group.num_pages == count and all(pool.shape[1] == count for pool in group.pools)
            assert all(entry.pages == count for entry in group.quantized)


def test_a_resize_whose_copies_fail_leaves_the_cache_as_it_was(kernels, monkeypatch):
    m = filled(None)
    before = [list(group.pools) for group in m.groups]
    copy, calls = kernels.copy_pages, [0]

    def second_fails(*args, **kwargs):
        calls[0] += 1
        if calls[0] == 2:
            raise KernelError("fails")
        copy(*args, **kwargs)

    monkeypatch.setattr(kernels, "copy_pages", second_fails)
    with pytest.raises(KernelError):
        m.resize(9)
    assert all(now is pool for group, pools in zip(m.groups, before) for now, pool in zip(group.pools, pools))
    m.check_consistency()
    write(m, "a", [8, 9])
    assert held(m, "a")[0] == list(range(1, 10)) and held(m, "c")[0] == [30, 31, 32]


# ------------------------------------------------------------------ the engine
@pytest.fixture
def tiny():
    return TinyEngine(*TINY["A"], torch.float32, "cpu")


def test_a_size_leaves_waiting_requests_room_beside_the_prefixes(tiny):
    """A prefix of three pages, a waiting request of five that does not start with it and one of five that does."""
    engine = engine_of(tiny, total_blocks=20, max_running_requests=1, max_prefixes=1)
    page = engine.manager.page_size
    tokens = random_prompt(tiny.config.vocab_size, 3 * page, 1)
    assert engine.add_prefix("p", tokens) == 3 * page
    prompts = {"first": random_prompt(tiny.config.vocab_size, 4, 2), "other": random_prompt(tiny.config.vocab_size, 5 * page - 6, 3),
               "sharing": tokens + random_prompt(tiny.config.vocab_size, 2 * page - 6, 4)}
    engine.submit("first", prompts["first"], max_new_tokens=3)
    engine.step()
    engine.submit("other", prompts["other"], max_new_tokens=6)
    engine.submit("sharing", prompts["sharing"], max_new_tokens=6, prefix="p")
    needs = engine.manager.lifetime_pages(engine.scheduler.get_request("other").lifetime_tokens)
    assert needs == (5,) and engine.manager.can_resize(7) == (7,)
    for size in (5, 7):
        with pytest.raises(OutOfPages, match="'other' could never be admitted"):
            engine.resize_cache(size)
        assert engine.manager.groups[0].num_pages == 20
    engine.resize_cache(8)
    engine.run()
    for name, prompt in prompts.items():
        assert list(engine.scheduler.get_request(name).generated_token_ids) == plain.greedy_tokens(
            tiny.tensors, tiny.config_dict, prompt, 3 if name == "first" else 6), name


def test_a_request_that_shares_a_prefix_needs_the_rest_of_its_pages(tiny):
    engine = engine_of(tiny, total_blocks=20, max_running_requests=1, max_prefixes=1)
    page = engine.manager.page_size
    tokens = random_prompt(tiny.config.vocab_size, 3 * page, 1)
    engine.add_prefix("p", tokens)
    prompt = tokens + random_prompt(tiny.config.vocab_size, 2 * page - 6, 4)
    engine.submit("sharing", prompt, max_new_tokens=6, prefix="p")
    with pytest.raises(OutOfPages):
        engine.resize_cache(4)
    engine.resize_cache(5)
    engine.run()
    assert list(engine.scheduler.get_request("sharing").generated_token_ids) == plain.greedy_tokens(tiny.tensors, tiny.config_dict, prompt, 6)
