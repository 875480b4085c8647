"""The rules of the requests on their logits, resident on the device and read by slot.

An engine made with ``logit_rules=True`` holds one set of tables (``ops.LogitTables``): penalties, the history of every slot's
tokens, biases and the tokens that a grammar allows.  Each step then applies them to the logits it samples from, in place, and
counts the tokens it chose, all on the device; a captured step finds whatever requests its rows belong to.  The host writes a
slot's rows when its request is admitted, and its grammar whenever the caller names other tokens.
"""

from __future__ import annotations

from collections.abc import Iterable, Sequence

import numpy as np
import torch

from .. import ops
from .params import SamplingParams


class LogitRules:
    """The tables of ``max_requests`` slots over ``vocab_size`` tokens (4.25 bytes per slot and token, 8 per bias of a slot)."""

    def __init__(self, max_requests: int, vocab_size: int, device: torch.device | str, *, max_biases: int = 300) -> None:
        if max_requests <= 0 or vocab_size <= 0 or max_biases < 0:
            raise ValueError("max_requests and vocab_size must be > 0, max_biases >= 0")
        self.vocab_size, self.max_biases, self.device = int(vocab_size), int(max_biases), torch.device(device)
        words = -(-vocab_size // 32)

        def table(width, fill, dtype=torch.int32):
            return torch.full((max_requests, width), fill, dtype=dtype, device=self.device)

        penalties = torch.tensor([1.0, 0.0, 0.0], device=self.device).repeat(max_requests, 1)
        self.tables = ops.LogitTables(penalties=penalties, counts=table(vocab_size, 0), seen=table(words, 0),
                                      bias_tokens=table(max_biases, ops.LogitTables.NO_TOKEN), bias_values=table(max_biases, 0.0, torch.float32),
                                      allowed=table(words, -1))

    def check(self, sampling: SamplingParams) -> None:
        if len(sampling.logit_bias) > self.max_biases:
            raise ValueError(f"{len(sampling.logit_bias)} biased tokens, the engine holds {self.max_biases} per request")
        if sampling.logit_bias and sampling.logit_bias[-1][0] >= self.vocab_size:
            raise ValueError(f"logit_bias names token {sampling.logit_bias[-1][0]} of a vocabulary of {self.vocab_size}")

    def _to_device(self, values, dtype: torch.dtype) -> torch.Tensor:
        return torch.tensor(values, dtype=dtype).to(self.device)

    def admit(self, slot: int, sampling: SamplingParams, prompt: Sequence[int]) -> None:
        """A new request owns the slot: its penalties and biases, its prompt as its history, every token allowed."""
        self.check(sampling)
        tables = self.tables
        tables.penalties[slot].copy_(self._to_device(
            [sampling.repetition_penalty, sampling.presence_penalty, sampling.frequency_penalty], torch.float32))
        tables.counts[slot].zero_()
        tables.seen[slot].zero_()
        tables.allowed[slot].fill_(-1)
        if self.max_biases:
            unused = self.max_biases - len(sampling.logit_bias)
            tables.bias_tokens[slot].copy_(self._to_device([t for t, _ in sampling.logit_bias] + [tables.NO_TOKEN] * unused, torch.int32))
            tables.bias_values[slot].copy_(self._to_device([v for _, v in sampling.logit_bias] + [0.0] * unused, torch.float32))
        tokens = self._to_device(list(prompt), torch.int32)
        ops.current().count_tokens(tokens, torch.full_like(tokens, slot), tables, prompt=True)

    def words_of(self, tokens: Iterable[int] | None) -> np.ndarray:
        """The given tokens (None: all) as the words of an ``allowed`` row."""
        words = -(-self.vocab_size // 32)
        if tokens is None:
            return np.full(words, -1, dtype=np.int32)
        index = np.fromiter(tokens, dtype=np.int64)
        if index.size and (index.min() < 0 or index.max() >= self.vocab_size):
            raise ValueError(f"allowed tokens must lie in [0, {self.vocab_size})")
        flags = np.zeros(words * 32, dtype=np.uint8)
        flags[index] = 1
        return np.packbits(flags, bitorder="little").view(np.int32)

    def allow(self, slot: int, words: np.ndarray) -> None:
        """The tokens that the slot's request may take from the next step on."""
        self.tables.allowed[slot].copy_(torch.from_numpy(words).to(self.device))
