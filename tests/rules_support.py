"""Rules on logits in plain Python, one request at a time, and the stand-ins of their kernels."""

from __future__ import annotations

import math

import torch

import plain_qwen2 as plain
from fake_ops import FakeOps
from mini_llm_runtime_b200.sampling import SamplingParams


def ruled(logits, sampling: SamplingParams, prompt, output, allowed=None):
    """One row of logits under a request's rules, entry by entry in 64 bits."""
    x = [float(v) for v in logits]
    for token in set(prompt) | set(output):
        x[token] = x[token] / sampling.repetition_penalty if x[token] > 0 else x[token] * sampling.repetition_penalty
    for token in set(output):
        x[token] -= sampling.frequency_penalty * list(output).count(token) + sampling.presence_penalty
    for token, value in sampling.logit_bias:
        x[token] += value
    if allowed is not None:
        x = [v if token in allowed else -math.inf for token, v in enumerate(x)]
    return torch.tensor(x, dtype=torch.float64)


def plain_run(tensors, config, sampling, prompt, count, allowed_after=None):
    """``count`` tokens by the plain implementation, greedy, the rules applied between; also the least distance between the two best
    logits of any step (a choice closer than rounding says nothing)."""
    output, gap = [], math.inf
    for _ in range(count):
        logits = plain.forward_logits(tensors, config, list(prompt) + output)[-1]
        allowed = None if allowed_after is None else allowed_after(output)
        x = ruled(logits, sampling, prompt, output, allowed)
        best = torch.topk(x, 2).values
        gap = min(gap, float(best[0] - best[1]))
        output.append(int(x.argmax()))
    return output, gap


class RuledFakeOps(FakeOps):
    """The stand-ins with those of the rules: the tables read by slot, as the kernels read them."""

    def shape_logits_(self, logits, row_slot, tables):
        vocab = logits.shape[1]
        for row, slot in enumerate(row_slot.tolist()):
            repetition, presence, frequency = tables.penalties[slot].tolist()
            for token in torch.nonzero(tables.counts[slot]).flatten().tolist():
                assert int(tables.seen[slot, token // 32]) >> (token % 32) & 1, "a known token has its bit"
                n = int(tables.counts[slot, token]) & (tables.IN_PROMPT - 1)
                x = float(logits[row, token])
                x = x / repetition if x > 0 else x * repetition
                logits[row, token] = x - frequency * n - presence * (n > 0)
            for token, value in zip(tables.bias_tokens[slot].tolist(), tables.bias_values[slot].tolist()):
                if token < vocab:
                    logits[row, token] += value
            for token in range(vocab):
                if not int(tables.allowed[slot, token // 32]) >> (token % 32) & 1:
                    logits[row, token] = -math.inf
        return logits

    def count_tokens(self, tokens, slots, tables, prompt=False):
        for token, slot in zip(tokens.tolist(), slots.tolist()):
            if prompt:
                tables.counts[slot, token] |= tables.IN_PROMPT
            else:
                tables.counts[slot, token] += 1
            word = int(tables.seen[slot, token // 32]) & 0xFFFFFFFF | 1 << (token % 32)
            tables.seen[slot, token // 32] = word - (1 << 32) if word >= 1 << 31 else word
