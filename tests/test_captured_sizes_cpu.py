"""What the step function remembers of the sizes it has met, without a device: which of them are to be captured, and how many."""

from __future__ import annotations

import pytest
import torch

from harness import TinyEngine
from mini_llm_runtime_b200 import ops
from mini_llm_runtime_b200.engine import StepEntry
from tiny_configs import TINY


@pytest.fixture
def runner(monkeypatch):
    runner = TinyEngine(*TINY["A"], torch.float32, "cpu").runner
    runner.use_graphs, runner.graph_capture_after = True, 3
    monkeypatch.setattr(ops, "_active", ops.CudaOps())
    return runner


def eligible(runner, monkeypatch, key):
    monkeypatch.setattr(runner, "_graph_key", lambda *args: key)
    return runner._graph_eligible([StepEntry("a", [1], [0])], [], True, False)


def test_sizes_of_groups_that_pass_by_are_forgotten(runner, monkeypatch):
    """A server whose prefixes' groups change size all the time: the memory of them stays bounded, a size that comes again is captured."""
    often = (4, True, False, 1024, (3, 48))
    for number in range(20000):
        assert not eligible(runner, monkeypatch, (4, True, False, 1024, (2, 16 * (number + 1)), (2, 16)))
        if number % 2000 == 0:
            assert eligible(runner, monkeypatch, often) == (number >= 4000)
    held = sum(len(value) for value in vars(runner).values() if isinstance(value, dict))
    assert held < 5000, held


def test_batch_sizes_are_counted_as_ever(runner, monkeypatch):
    for count in range(1, 200):
        for expected in (False, False, True, True):
            assert eligible(runner, monkeypatch, (count, True, False, 1024)) == expected
    for number in range(5000):
        eligible(runner, monkeypatch, (4, True, False, 1024, (2, 16 * (number + 1))))
    assert eligible(runner, monkeypatch, (1, True, False, 1024))
