"""Draws with a temperature from rows in which most tokens are forbidden (their logits -inf, as grammars and bans leave them): a
token of no probability never comes out, wherever the sums of the probabilities are rounded."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from mini_llm_runtime_b200 import ops

pytestmark = pytest.mark.gpu

DEVICE = "cuda:0"
WARPS = 32                # stretches of the vocabulary that are summed by themselves, then walked


def uniforms(seed: int, count: int) -> np.ndarray:
    """The sampler's generator for counters 0 .. count - 1, as whole numbers of 2^-24."""
    with np.errstate(over="ignore"):
        z = np.uint64(seed) + np.arange(1, count + 1, dtype=np.uint64) * np.uint64(0x9E3779B97F4A7C15)
        z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
        z = z ^ (z >> np.uint64(31))
    return (z >> np.uint64(40)).astype(np.int64)


def draw(row, counters, temperature=1.0, seed=3):
    """One token per counter from the same row."""
    rows = len(counters)
    logits = row.to(DEVICE).expand(rows, -1).contiguous()
    return ops.current().sample(logits, torch.full((rows,), float(temperature), device=DEVICE),
                                torch.full((rows,), seed, dtype=torch.int64, device=DEVICE),
                                torch.as_tensor(counters, dtype=torch.int64, device=DEVICE)).cpu()


@pytest.mark.parametrize("vocab", [32768, 65536])
def test_a_target_that_the_walk_does_not_reach(vocab):
    """All tokens of the first 31 stretches weigh one; the last stretch has one token in each 32, too light to be seen beside the
    31 stretches' sum (less than half a step of float32), though together they have weight.  A draw that falls to the last stretch finds
    no token at which the running sum passes it: it takes one of the stretch's allowed tokens."""
    stretch = vocab // WARPS
    head = (WARPS - 1) * stretch
    step = 2.0 ** (math.floor(math.log2(head)) - 23)
    light = 0.49 * step
    row = torch.zeros(vocab)
    row[head:] = -math.inf
    row[head + 7::32] = math.log(light)
    # Draws past the head's share by at least two steps, and no others: u (head + sum of the light ones) rounds to such a number.
    total = np.float32(head) + np.float32(light * (stretch // 32))
    numbers = uniforms(3, 1 << 25)
    target = (numbers.astype(np.float32) * np.float32(2.0 ** -24) * total).astype(np.float32)
    counters = np.nonzero(target >= head + 2 * step)[0][:64]
    assert len(counters) >= 8, "the case must meet the last stretch"
    tokens = draw(row, counters)
    assert bool((row[tokens.long()] > -math.inf).all()), tokens.tolist()
    assert int(tokens.min()) >= head


@pytest.mark.parametrize("vocab", [40, 1000, 32003, 152064])
@pytest.mark.parametrize("temperature", [0.05, 1.0, 7.0])
def test_a_single_allowed_token(vocab, temperature):
    """In the middle of a stretch, in its first and its last place."""
    stretch = ((vocab + WARPS - 1) // WARPS + 31) // 32 * 32
    for token in sorted({0, stretch // 2, stretch - 1, min(vocab - 1, stretch), vocab // 2, vocab - 2}):
        row = torch.full((vocab,), -math.inf)
        row[token] = -3.0
        assert draw(row, range(100), temperature).unique().tolist() == [token]


@pytest.mark.parametrize("vocab", [1000, 32003])
def test_few_allowed_tokens(vocab):
    """Random grammars of a few tokens, weights over twelve powers of ten: every draw is allowed."""
    g = torch.Generator().manual_seed(vocab)
    for _ in range(20):
        allowed = torch.randperm(vocab, generator=g)[:7]
        row = torch.full((vocab,), -math.inf)
        row[allowed] = torch.rand(7, generator=g) * 27.6 - 30
        tokens = draw(row, range(1000))
        assert bool(torch.isin(tokens.long(), allowed).all())


def test_shares_of_allowed_tokens():
    """Three tokens of weights 1, 2 and 5 beside forbidden ones, 8,000 draws: counts within five standard deviations."""
    vocab = 5000
    row = torch.full((vocab,), -math.inf)
    places, weights = [17, 2600, 4998], [1.0, 2.0, 5.0]
    row[places] = torch.tensor(weights).log()
    count = 8000
    tokens = torch.cat([draw(row, range(start, start + 1000)) for start in range(0, count, 1000)])
    for place, weight in zip(places, weights):
        share = weight / sum(weights)
        assert abs(int((tokens == place).sum()) - share * count) < 5 * math.sqrt(count * share * (1 - share))


@pytest.mark.parametrize("vocab", [40, 1000, 152064])
@pytest.mark.parametrize("temperature", [0.0, 0.05, 1.0, 7.0])
def test_a_row_that_allows_nothing(vocab, temperature):
    """Token 0 at any temperature."""
    assert not draw(torch.full((vocab,), -math.inf), range(20), temperature).any()


@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_an_infinite_logit_is_the_choice(temperature):
    row = torch.full((1000,), -math.inf)
    row[::3] = torch.linspace(-5, 5, 334)
    row[333] = math.inf
    assert draw(row, range(20), temperature).unique().tolist() == [333]


@pytest.mark.parametrize("vocab", [1000, 1003, 32000])
@pytest.mark.parametrize("entries", [0, 1, 2, 3])
def test_logits_on_any_boundary(vocab, entries):
    """A view into a larger tensor: the same tokens as from a tensor of its own, greedy and drawn."""
    rows = 5
    g = torch.Generator().manual_seed(vocab)
    logits = torch.randn((rows, vocab), generator=g).to(DEVICE)
    view = torch.empty(rows * vocab + 8, device=DEVICE)[entries:entries + rows * vocab].view(rows, vocab)
    view.copy_(logits)
    for temperature in (0.0, 1.0):
        options = (torch.full((rows,), temperature, device=DEVICE), torch.arange(rows, device=DEVICE), torch.arange(rows, device=DEVICE))
        got = ops.current().sample(view, *options)
        assert torch.equal(got, ops.current().sample(logits, *options))
        if temperature == 0:
            assert torch.equal(got.long(), logits.argmax(dim=1))
