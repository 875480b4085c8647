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
