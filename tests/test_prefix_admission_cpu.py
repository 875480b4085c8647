"""Requests beside prefixes that the cache keeps: what the prefixes leave of the pool decides what can ever be admitted, when a request
is submitted and when a prefix is added, so that no request waits for room that will not come."""

from __future__ import annotations

import pytest
import torch

import plain_qwen2 as plain
from harness import TinyEngine, random_prompt
from mini_llm_runtime_b200 import ops
from mini_llm_runtime_b200.cache import OutOfPages
from mini_llm_runtime_b200.engine import ContinuousBatchEngine
from mini_llm_runtime_b200.ops import cuda_ops
from test_cache_manager import manager
from test_shared_pages_cpu import SharedFakeOps
from tiny_configs import TINY

PAGE = TINY["A"][1]


@pytest.fixture(autouse=True)
def kernels(monkeypatch):
    monkeypatch.setattr(cuda_ops, "_need", lambda *args, **kwargs: None)
    with ops.use(SharedFakeOps()) as stand_in:
        yield stand_in


@pytest.fixture
def tiny():
    return TinyEngine(*TINY["A"], torch.float32, "cpu")


def engine_of(tiny, pages):
    return ContinuousBatchEngine.from_model(tiny.model, block_size=PAGE, total_blocks=pages, max_running_requests=3, max_batch_tokens=24,
                                            max_model_len=160, max_prefixes=2)


def finished(engine, tiny, name, prompt, count):
    want = plain.greedy_tokens(tiny.tensors, tiny.config_dict, prompt, count)
    return list(engine.scheduler.get_request(name).generated_token_ids) == want


def test_a_request_that_the_prefixes_leave_no_room_for(tiny):
    """Ten pages, six of them a prefix's: a request of five pages of its own is refused, one of four is served."""
    engine = engine_of(tiny, 10)
    vocab = tiny.config.vocab_size
    prefix = random_prompt(vocab, 6 * PAGE, 1)
    engine.add_prefix("p", prefix)
    with pytest.raises(ValueError, match="never be admitted"):
        engine.submit("a", random_prompt(vocab, 4 * PAGE, 2), max_new_tokens=2)
    shares_one = prefix[:PAGE] + [prefix[PAGE] ^ 1] + random_prompt(vocab, 5 * PAGE, 3)
    with pytest.raises(ValueError, match="does not start"):
        engine.submit("b", shares_one, max_new_tokens=2, prefix="p")
    short = prefix[:PAGE + 1]                              # shares one page; its own tokens fill five
    with pytest.raises(ValueError, match="never be admitted"):
        engine.submit("c", short, max_new_tokens=5 * PAGE, prefix="p")
    prompts = {"d": random_prompt(vocab, 4 * PAGE, 4), "e": short, "f": prefix + [1]}
    engine.submit("d", prompts["d"], max_new_tokens=1)
    engine.submit("e", prompts["e"], max_new_tokens=4 * PAGE, prefix="p")      # one shared and four of its own
    engine.submit("f", prompts["f"], max_new_tokens=3 * PAGE, prefix="p")
    engine.run()
    assert finished(engine, tiny, "d", prompts["d"], 1) and finished(engine, tiny, "e", prompts["e"], 4 * PAGE)
    assert finished(engine, tiny, "f", prompts["f"], 3 * PAGE)
    engine.drop_prefix("p")
    engine.submit("a", random_prompt(vocab, 4 * PAGE, 2), max_new_tokens=2)     # nothing is held any more
    engine.run()
    engine.manager.check_consistency()


def test_a_prefix_that_would_shut_a_waiting_request_out(tiny):
    engine = engine_of(tiny, 10)
    vocab = tiny.config.vocab_size
    long = random_prompt(vocab, 6 * PAGE, 1)
    engine.submit("long", long, max_new_tokens=2)          # seven pages, still waiting
    with pytest.raises(OutOfPages, match="'long'"):
        engine.add_prefix("p", random_prompt(vocab, 4 * PAGE, 2))
    assert engine.manager.stats().live_requests == 0
    engine.add_prefix("q", random_prompt(vocab, 3 * PAGE, 3))
    engine.run()
    assert finished(engine, tiny, "long", long, 2)
    engine.add_prefix("p", random_prompt(vocab, 4 * PAGE, 2))
    engine.manager.check_consistency()


def test_two_prefixes_count_together(tiny):
    engine = engine_of(tiny, 10)
    vocab = tiny.config.vocab_size
    prefixes = [random_prompt(vocab, 4 * PAGE, seed) for seed in (1, 2)]
    for name, tokens in zip("pq", prefixes):
        engine.add_prefix(name, tokens)
    for name, prompt, prefix in (("a", random_prompt(vocab, 2 * PAGE, 3), None), ("b", prefixes[0] + random_prompt(vocab, 2 * PAGE, 4), "p")):
        with pytest.raises(ValueError, match="never be admitted"):
            engine.submit(name, prompt, max_new_tokens=2, prefix=prefix)
        engine.submit(name + "1", prompt[:-1], max_new_tokens=2, prefix=prefix)
    engine.run()
    assert finished(engine, tiny, "b1", prefixes[0] + random_prompt(vocab, 2 * PAGE, 4)[:-1], 2)


def test_prefixes_that_do_not_fit(tiny):
    engine = engine_of(tiny, 8)
    vocab = tiny.config.vocab_size
    with pytest.raises(ValueError, match="never be admitted"):
        engine.add_prefix("p", random_prompt(vocab, 9 * PAGE, 1))      # more than the pool
    engine.add_prefix("p", random_prompt(vocab, 5 * PAGE, 1))
    with pytest.raises(OutOfPages, match="no room"):
        engine.add_prefix("q", random_prompt(vocab, 4 * PAGE, 2))      # more than the first one leaves
    engine.add_prefix("q", random_prompt(vocab, 3 * PAGE, 2))
    engine.manager.check_consistency()


def test_the_manager_by_itself():
    m = manager(pages=8, page=4)
    m.create_request("kept", lifetime_tokens=12, lasting=True)
    m.begin_step([("kept", 12)])
    m.commit_step()
    assert m.can_be_admitted(20) and not m.can_be_admitted(21)
    assert m.can_be_admitted(28, ("kept", 8)) and not m.can_be_admitted(29, ("kept", 8))
    assert m.can_be_admitted(20, beside=0) and not m.can_be_admitted(20, beside=1) and m.can_be_admitted(16, beside=4)
    for lifetime, prefix in ((21, None), (29, ("kept", 8))):
        with pytest.raises(ValueError, match="never be admitted"):
            m.create_request("a", lifetime_tokens=lifetime, prefix=prefix)
    # pages of a request that ends by itself are only held as long as those that share them
    m.create_request("b", lifetime_tokens=9)
    m.begin_step([("b", 9)])
    m.commit_step()
    assert m.can_be_admitted(20, ("b", 8)) and not m.can_be_admitted(21, ("b", 8))
    assert m.create_request("c", lifetime_tokens=17, prefix=("b", 8)) is None       # three pages of its own, two are left: it may wait
    assert m.create_request("c", lifetime_tokens=16, prefix=("b", 8)) is not None
    m.check_consistency()
    m.release("c")
    m.release("b")
    m.release("kept")
    assert m.can_be_admitted(32) and m.create_request("d", lifetime_tokens=32) is not None
