"""Which parts take a cache in 8 bits, said when the engine is made."""

from __future__ import annotations

import pytest
import torch

import toy_parts
from harness import TinyEngine
from mini_llm_runtime_b200.config.spec import PartSpec
from mini_llm_runtime_b200.ops import cuda_ops
from mini_llm_runtime_b200.parts.base import build_part
from test_forked_requests_cpu import engine_of
from tiny_configs import TINY


def attention(position):
    return build_part("mixer", PartSpec("gqa_attention", {"hidden_size": 64, "num_heads": 4, "num_kv_heads": 2, "head_dim": 16,
                                                          "position": position}, "x."), torch.float32)


def test_attention_with_an_encoding_that_stores_its_keys_itself_refuses_a_cache_in_8_bits(monkeypatch):
    monkeypatch.setattr(cuda_ops, "_need", lambda *args, **kwargs: None)
    toy_parts.register_toys()
    assert attention(None).supports_quantized_cache
    assert not attention(PartSpec("toy_no_rotation", {"head_dim": 16})).supports_quantized_cache
    tiny = TinyEngine(*TINY["A"], torch.float32, "cpu")
    assert all(block.mixer.supports_quantized_cache for block in tiny.model.blocks)
    tiny.model.blocks[1].mixer = attention(PartSpec("toy_no_rotation", {"head_dim": 16}))
    engine_of(tiny)
    with pytest.raises(ValueError, match="8 bits"):
        engine_of(tiny, cache_dtype="int8")
