"""A grammar that was named for a request before it ran goes with the request, however that ends."""

from __future__ import annotations

import pytest

from harness import random_prompt
from mini_llm_runtime_b200.ops import KernelError, current
from test_logit_rules_engine_cpu import engine_of, stand_in_kernels, tiny  # noqa: F401  (fixtures)


@pytest.mark.parametrize("length", [9, 60])
def test_a_request_that_ends_with_an_error(tiny, length):  # noqa: F811
    """In the step of its first token, or in a portion of its prompt before that."""
    vocab = tiny.config.vocab_size
    engine = engine_of(tiny)
    engine.submit("a", random_prompt(vocab, length, 1), max_new_tokens=3)
    engine.allow_tokens("a", [3, 4])
    engine.submit("b", random_prompt(vocab, 9, 2), max_new_tokens=3)
    engine.allow_tokens("b", [5])
    current().error_code = 3
    with pytest.raises(KernelError):
        engine.step()
    assert engine.scheduler.get_request("a").finish_reason.value == "error"
    assert "a" not in engine._allowed
    engine.run()
    assert not engine._allowed
    if length == 60:                    # the second request had not begun, and keeps its grammar
        assert list(engine.scheduler.get_request("b").generated_token_ids)[0] == 5
