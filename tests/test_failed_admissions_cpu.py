"""Admissions that fail half-way: what the cache manager and the scheduler hold afterwards is what they held before."""

from __future__ import annotations

import pytest
import torch

import plain_qwen2 as plain
from harness import TinyEngine, random_prompt
from mini_llm_runtime_b200 import ops
from mini_llm_runtime_b200.ops import KernelError, cuda_ops
from requests_support import RequestFakeOps
from test_forked_requests_cpu import engine_of, held, manager, write
from tiny_configs import TINY


@pytest.fixture(autouse=True)
def kernels(monkeypatch):
    monkeypatch.setattr(cuda_ops, "_need", lambda *args, **kwargs: None)
    with ops.use(RequestFakeOps()) as stand_in:
        yield stand_in


def failing_copies(kernels, monkeypatch, which):
    """The ``which``-th call of copy_pages from now on raises."""
    copy, calls = kernels.copy_pages, [0]

    def some(*args, **kwargs):
        calls[0] += 1
        if calls[0] == which:
            raise KernelError("the copy fails")
        copy(*args, **kwargs)

    monkeypatch.setattr(kernels, "copy_pages", some)


@pytest.mark.parametrize("options", [{}, {"lifetime_tokens": 16}])
@pytest.mark.parametrize("which", [1, 2])
def test_a_fork_whose_copy_fails_holds_nothing(which, options, kernels, monkeypatch):
    m = manager(pages=12, page=4)
    m.create_request("a")
    write(m, "a", list(range(1, 11)))
    before, free_slots = m.stats(), m.slots.free_count
    failing_copies(kernels, monkeypatch, which)
    with pytest.raises(KernelError):
        m.create_request("b", fork=("a", 10), **options)
    assert m.stats() == before and m.slots.free_count == free_slots and "b" not in m.requests
    assert not any(group.borrowers for group in m.groups)
    m.check_consistency()
    m.create_request("b", fork=("a", 10), **options)       # the calls after it do not fail
    assert held(m, "b")[0] == list(range(1, 11))
    m.release("a")
    m.release("b")
    m.check_consistency()
    assert m.stats().free_pages == (12,) * len(m.groups) and m.stats().promised_pages == (0,) * len(m.groups)


# ------------------------------------------------------------------ the engine
@pytest.fixture
def tiny():
    return TinyEngine(*TINY["A"], torch.float32, "cpu")


@pytest.mark.parametrize("step_ahead", [False, True])
def test_requests_admitted_before_one_that_fails_are_admitted_again(step_ahead, tiny, kernels, monkeypatch):
    """Two requests with limits of their own and a fork in one planning; the fork's copy fails.  The next planning admits them all, limits included."""
    engine = engine_of(tiny, sampling_limits=True, step_ahead=step_ahead)
    prompt = random_prompt(tiny.config.vocab_size, 30, 3)
    other = random_prompt(tiny.config.vocab_size, 11, 4)
    engine.submit("a", prompt, max_new_tokens=8)
    engine.step()
    engine.submit("one", other, max_new_tokens=5, temperature=3.0, top_k=1)
    engine.submit("sure", other, max_new_tokens=5, temperature=3.0, min_p=1.0)
    engine.submit("fork", prompt, max_new_tokens=4, fork_of="a")
    failing_copies(kernels, monkeypatch, 1)
    with pytest.raises(KernelError):
        engine.step()
    assert engine.scheduler.running_request_ids == ("a",) and engine.scheduler.waiting_request_ids == ("one", "sure", "fork")
    assert engine.scheduler.outstanding_plan is None and set(engine.manager.requests) == {"a"}
    engine.manager.check_consistency()
    engine.run()
    for name, text, count in (("a", prompt, 8), ("one", other, 5), ("sure", other, 5), ("fork", prompt, 4)):
        assert list(engine.scheduler.get_request(name).generated_token_ids) == plain.greedy_tokens(tiny.tensors, tiny.config_dict, text, count), name
    assert engine.manager.stats().free_pages == (40,) and engine.manager.stats().promised_pages == (0,)


def test_a_fork_given_back_is_planned_by_its_whole_prompt(tiny, monkeypatch):
    """Without portions of prompts a request runs in one step or waits: what a fork shared in a step that failed counts no more when its
    other request has ended."""
    engine = engine_of(tiny, chunked_prefill=False, max_batch_tokens=34)
    prompt = random_prompt(tiny.config.vocab_size, 33, 5)
    engine.submit("a", prompt, max_new_tokens=2)
    engine.step()
    engine.submit("b", prompt, max_new_tokens=2, fork_of="a")
    forward = engine.runner.model.forward
    monkeypatch.setattr(engine.runner.model, "forward", lambda ctx: (_ for _ in ()).throw(RuntimeError("fails")))
    with pytest.raises(RuntimeError, match="fails"):
        engine.step()
    monkeypatch.setattr(engine.runner.model, "forward", forward)
    request = engine.scheduler.get_request("b")
    assert (request.shared, request.cursor) == (0, 0) and engine.scheduler.waiting_request_ids == ("b",)
    engine.scheduler.fail_requests(["a"])
    engine.submit("c", random_prompt(tiny.config.vocab_size, 5, 6), max_new_tokens=8)
    engine.run()
    assert list(request.generated_token_ids) == plain.greedy_tokens(tiny.tensors, tiny.config_dict, prompt, 2)
