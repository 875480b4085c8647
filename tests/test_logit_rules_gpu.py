"""The rules of requests on their logits (``shape_logits``, ``shape_logits_``, ``count_tokens``) against their definition in 64
bits, written here entry by entry, at vocabularies that no vector width divides and with tables that leave a row empty."""

from __future__ import annotations

import math

import pytest
import torch

from mini_llm_runtime_b200 import ops
from mini_llm_runtime_b200.ops import LogitTables

pytestmark = pytest.mark.gpu

DEVICE = "cuda:0"
HALF_STEP = torch.finfo(torch.float32).eps / 2


def bits(flags):
    """Truth values [n, width] as words, by the definition: token t in bit t % 32 of word t // 32."""
    words = torch.zeros((flags.shape[0], -(-flags.shape[1] // 32)), dtype=torch.int64)
    for row, token in torch.nonzero(flags).tolist():
        words[row, token // 32] |= 1 << (token % 32)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def made(vocab, slots, seed, *, penalties=True, biases=0, grammar=False, known=0.2):
    """Tables on the CPU: histories, biases with a token listed twice, a grammar under which slot 0 allows nothing."""
    g = torch.Generator().manual_seed(seed)
    out = {}
    if penalties:
        counts = torch.randint(1, 6, (slots, vocab), generator=g, dtype=torch.int32)
        counts[torch.rand((slots, vocab), generator=g) < 0.5] |= LogitTables.IN_PROMPT
        only = torch.rand((slots, vocab), generator=g) < 0.3
        counts[only] = LogitTables.IN_PROMPT
        counts[torch.rand((slots, vocab), generator=g) >= known] = 0
        out["counts"] = counts
        out["seen"] = bits(counts != 0)
        out["penalties"] = torch.stack([0.6 + torch.rand(slots, generator=g), torch.rand(slots, generator=g) * 2 - 0.5,
                                        torch.rand(slots, generator=g)], dim=1).contiguous()
    if biases:
        tokens = torch.randint(0, vocab, (slots, biases), generator=g).sort(dim=1).values
        if biases > 2:
            tokens[:, 1] = tokens[:, 0]
            tokens[:, -1] = LogitTables.NO_TOKEN
        out["bias_tokens"] = tokens.to(torch.int32)
        out["bias_values"] = torch.randn((slots, biases), generator=g) * 5
    if grammar:
        allowed = torch.rand((slots, vocab), generator=g) < 0.5
        allowed[0] = False
        out["allowed"] = bits(allowed)
    return out


def exact(logits, row_slot, tables):
    """The definition, and per entry the sum of magnitudes that its roundings are relative to."""
    x = logits.double().clone()
    size = x.abs().clone()
    vocab = x.shape[1]
    for row, slot in enumerate(row_slot.tolist()):
        slots = next(t.shape[0] for t in tables.values())
        if not 0 <= slot < slots:
            continue
        if "counts" in tables:
            repetition, presence, frequency = (float(p) for p in tables["penalties"][slot])
            word = tables["counts"][slot]
            known = word != 0
            n = (word & (LogitTables.IN_PROMPT - 1)).double()
            x[row] = torch.where(known, torch.where(x[row] > 0, x[row] / repetition, x[row] * repetition), x[row])
            size[row] = torch.maximum(size[row], x[row].abs()) + abs(frequency) * n + abs(presence) * (n > 0)
            x[row] -= frequency * n + presence * (n > 0)
        if "bias_tokens" in tables:
            for token, value in zip(tables["bias_tokens"][slot].tolist(), tables["bias_values"][slot].tolist()):
                if 0 <= token < vocab:
                    x[row, token] += value
                    size[row, token] += abs(value)
        if "allowed" in tables:
            words = tables["allowed"][slot].long() & 0xFFFFFFFF
            index = torch.arange(vocab)
            x[row][(words[index // 32] >> (index % 32)) & 1 == 0] = -math.inf
    return x, size


def check(got, logits, row_slot, tables, most_biases):
    want, size = exact(logits, row_slot, tables)
    got = got.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    solid = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), solid)
    odd = ~solid & ~torch.isnan(want)
    assert torch.equal(got[odd], want[odd])
    # one rounding each: the repetition, frequency * n, two differences, each further bias of a token and its addition
    roundings = 5 + most_biases
    bound = roundings * HALF_STEP * size * (1 + 1e-6)
    assert bool(((got - want).abs() <= bound)[solid].all()), float(((got - want).abs() - bound)[solid].max())


def on_device(tables):
    return LogitTables(**{name: tensor.to(DEVICE) for name, tensor in tables.items()})


@pytest.mark.parametrize("rules", ["penalties", "biases", "grammar", "all"])
@pytest.mark.parametrize("vocab", [1, 3, 5, 32, 33, 127, 1000, 4093, 4096, 4097, 32003])
def test_rules_against_their_definition(vocab, rules):
    slots, rows = 5, 7
    g = torch.Generator().manual_seed(vocab)
    logits = torch.randn((rows, vocab), generator=g) * 4
    row_slot = torch.tensor([3, 0, 4, 4, -1, 5, 1], dtype=torch.int32)      # two rows of one slot, two of none
    biases = min(9, vocab) if rules in ("biases", "all") else 0
    tables = made(vocab, slots, vocab + 1, penalties=rules in ("penalties", "all"), biases=biases, grammar=rules in ("grammar", "all"))
    device = on_device(tables)
    most = 2 + biases if vocab < 40 else 4
    got = ops.current().shape_logits(logits.to(DEVICE), row_slot.to(DEVICE), device)
    check(got, logits, row_slot, tables, most)
    assert torch.equal(got[4:6].cpu(), logits[4:6]), "a row of no slot passes unchanged"
    if rules in ("grammar", "all"):
        assert bool((got[1] == -math.inf).all()), "slot 0 allows nothing"
        assert int(ops.current().sample(got, torch.zeros(rows, device=DEVICE), torch.zeros(rows, dtype=torch.int64, device=DEVICE),
                                        torch.zeros(rows, dtype=torch.int64, device=DEVICE))[1]) == 0
    placed = logits.to(DEVICE)
    same = ops.current().shape_logits_(placed, row_slot.to(DEVICE), device)
    assert same is placed and torch.equal(placed, got), "in place and out of place are the same arithmetic"


@pytest.mark.parametrize("rows,vocab", [(1, 151936), (70, 20011)])
def test_large_rows(rows, vocab):
    g = torch.Generator().manual_seed(rows)
    logits = torch.randn((rows, vocab), generator=g) * 4
    row_slot = torch.randperm(rows, generator=g).to(torch.int32)
    tables = made(vocab, rows, rows + 1, biases=600, grammar=False, known=0.01)
    tables["allowed"] = torch.randint(-(1 << 31), 1 << 31, (rows, -(-vocab // 32)), generator=g).to(torch.int32)
    got = ops.current().shape_logits(logits.to(DEVICE), row_slot.to(DEVICE), on_device(tables))
    check(got, logits, row_slot, tables, 6)


def test_infinities_and_nan_in_logits():
    vocab = 37
    logits = torch.randn((2, vocab), generator=torch.Generator().manual_seed(5))
    logits[:, 3], logits[:, 4], logits[:, 5] = math.inf, -math.inf, math.nan
    logits[:, 6], logits[:, 7], logits[:, 8] = math.inf, -math.inf, math.nan
    logits[:, 9], logits[:, 10] = torch.finfo(torch.float32).min, 0.0
    tables = made(vocab, 2, 6, biases=5, known=1.0)
    allowed = torch.ones((2, vocab), dtype=torch.bool)
    allowed[:, 6:9] = False
    tables["allowed"] = bits(allowed)
    tables["penalties"][:, 0] = 0.9       # the lowest value times the repetition stays finite
    row_slot = torch.tensor([0, 1], dtype=torch.int32)
    got = ops.current().shape_logits(logits.to(DEVICE), row_slot.to(DEVICE), on_device(tables))
    check(got, logits, row_slot, tables, 5)
    assert bool((got[:, 6:9] == -math.inf).all()), "what stands in a forbidden place is not looked at"


def test_a_ban_by_a_bias_of_minus_infinity():
    tables = {"bias_tokens": torch.tensor([[2, 5]], dtype=torch.int32), "bias_values": torch.tensor([[-math.inf, 1.5]])}
    got = ops.current().shape_logits(torch.ones((1, 8), device=DEVICE), torch.zeros(1, dtype=torch.int32, device=DEVICE), on_device(tables))
    assert got[0].tolist() == [1, 1, -math.inf, 1, 1, 2.5, 1, 1]


def test_no_rows_and_no_biases():
    tables = made(100, 2, 3)
    tables["bias_tokens"], tables["bias_values"] = torch.zeros((2, 0), dtype=torch.int32), torch.zeros((2, 0))
    kernels = ops.current()
    none = kernels.shape_logits(torch.empty((0, 100), device=DEVICE), torch.empty(0, dtype=torch.int32, device=DEVICE), on_device(tables))
    assert none.shape == (0, 100)
    logits = torch.randn((1, 100), generator=torch.Generator().manual_seed(1))
    got = kernels.shape_logits(logits.to(DEVICE), torch.ones(1, dtype=torch.int32, device=DEVICE), on_device(tables))
    check(got, logits, torch.ones(1, dtype=torch.int32), tables, 0)


def test_history_grows_by_tokens():
    vocab, slots = 1003, 4
    device = LogitTables(penalties=torch.tensor([[1.3, 0.4, 0.2]] * slots, device=DEVICE),
                         counts=torch.zeros((slots, vocab), dtype=torch.int32, device=DEVICE),
                         seen=torch.zeros((slots, 32), dtype=torch.int32, device=DEVICE))
    g = torch.Generator().manual_seed(9)
    want = torch.zeros((slots, vocab), dtype=torch.int64)
    kernels = ops.current()
    for prompt in (True, False, False):
        tokens = torch.randint(-2, vocab + 2, (500,), generator=g, dtype=torch.int32)
        tokens[:100] = 1002                   # one token many times
        owners = torch.randint(-1, slots + 1, (500,), generator=g, dtype=torch.int32)
        kernels.count_tokens(tokens.to(DEVICE), owners.to(DEVICE), device, prompt=prompt)
        for token, slot in zip(tokens.tolist(), owners.tolist()):
            if 0 <= token < vocab and 0 <= slot < slots:
                want[slot, token] = want[slot, token] | LogitTables.IN_PROMPT if prompt else want[slot, token] + 1
    assert torch.equal(device.counts.cpu().long(), want)
    assert torch.equal(device.seen.cpu(), bits(want != 0))
    kernels.count_tokens(torch.empty(0, dtype=torch.int32, device=DEVICE), torch.empty(0, dtype=torch.int32, device=DEVICE), device)


def test_a_captured_step_follows_its_tables():
    """Rules, choice and history as a decode step runs them, captured once and replayed while the tables change."""
    vocab, slots, rows = 4099, 3, 2
    kernels = ops.current()
    tables = made(vocab, slots, 12, biases=4, grammar=False)
    device = on_device(tables)
    logits = (torch.randn((rows, vocab), generator=torch.Generator().manual_seed(2))).to(DEVICE)
    row_slot = torch.tensor([2, 0], dtype=torch.int32, device=DEVICE)
    zero = torch.zeros(rows, dtype=torch.int64, device=DEVICE)
    cold = torch.zeros(rows, device=DEVICE)

    def step():
        shaped = kernels.shape_logits(logits, row_slot, device)
        tokens = kernels.sample(shaped, cold, zero, zero)
        kernels.count_tokens(tokens, row_slot, device)
        return shaped, tokens

    before = device.counts.clone(), device.seen.clone()
    step()
    torch.cuda.synchronize()
    device.counts.copy_(before[0]), device.seen.copy_(before[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        shaped, tokens = step()
    for turn in range(4):
        row_slot.copy_(torch.tensor([[2, 0], [1, 2], [1, 0], [2, 0]][turn], dtype=torch.int32))
        now = {"counts": device.counts.cpu(), "seen": device.seen.cpu(), "penalties": tables["penalties"],
               "bias_tokens": tables["bias_tokens"], "bias_values": tables["bias_values"]}
        graph.replay()
        torch.cuda.synchronize()
        check(shaped, logits.cpu(), row_slot.cpu(), now, 4)
        assert torch.equal(tokens.cpu().long(), shaped.cpu().argmax(dim=1))
        for slot, token in zip(row_slot.tolist(), tokens.tolist()):
            now["counts"][slot, token] += 1
        assert torch.equal(device.counts.cpu(), now["counts"])
        assert torch.equal(device.seen.cpu(), bits(now["counts"] != 0))


def test_on_another_stream():
    tables = made(2048, 1, 3, biases=3)
    logits = torch.randn((1, 2048), generator=torch.Generator().manual_seed(4))
    device, slot = on_device(tables), torch.zeros(1, dtype=torch.int32, device=DEVICE)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = ops.current().shape_logits(logits.to(DEVICE), slot, device)
    stream.synchronize()
    check(got, logits, torch.zeros(1, dtype=torch.int32), tables, 3)


def test_history_words_beyond_32_bit_offsets():
    vocab = 151936
    slots = (1 << 31) // vocab + 3            # the last slots' words lie more than 2^31 entries in
    kernels = ops.current()
    device = LogitTables(penalties=torch.tensor([[2.0, 0.5, 0.25]], device=DEVICE).repeat(slots, 1),
                         counts=torch.zeros((slots, vocab), dtype=torch.int32, device=DEVICE),
                         seen=torch.zeros((slots, -(-vocab // 32)), dtype=torch.int32, device=DEVICE))
    last = torch.tensor([slots - 1, slots - 1], dtype=torch.int32, device=DEVICE)
    kernels.count_tokens(torch.tensor([vocab - 1, vocab - 1], dtype=torch.int32, device=DEVICE), last, device)
    logits = torch.ones((1, vocab), device=DEVICE)
    got = kernels.shape_logits(logits, last[:1], device)
    want = torch.ones((1, vocab))
    want[0, vocab - 1] = 0.5 - 0.5 - 0.5
    assert torch.equal(got.cpu(), want)
    assert int(device.counts.sum()) == 2


def test_logits_on_no_16_byte_boundary_are_refused():
    tables = on_device(made(31, 2, 3))
    logits = torch.zeros((2, 31), device=DEVICE)[1:]
    with pytest.raises(ops.KernelError, match="aligned"):
        ops.current().shape_logits(logits, torch.zeros(1, dtype=torch.int32, device=DEVICE), tables)
