"""Rules on logits whose tables are views into larger ones: on any boundary that their entries may have."""

from __future__ import annotations

import pytest
import torch

from mini_llm_runtime_b200 import ops
from mini_llm_runtime_b200.ops import LogitTables
from test_logit_rules_gpu import check, made

pytestmark = pytest.mark.gpu

DEVICE = "cuda:0"


def both_ways(logits, row_slot, device):
    """The same logits apart and in place."""
    got = ops.current().shape_logits(logits.to(DEVICE), row_slot.to(DEVICE), device)
    placed = logits.to(DEVICE)
    assert torch.equal(ops.current().shape_logits_(placed, row_slot.to(DEVICE), device), got)
    return got


def moved(tensor, entries):
    """A copy on the device that starts so many entries behind a boundary of 256 bytes."""
    room = torch.empty(tensor.numel() + 64, dtype=tensor.dtype, device=DEVICE)
    view = room[entries:entries + tensor.numel()].view(tensor.shape)
    return view.copy_(tensor)


@pytest.mark.parametrize("vocab", [5, 1000, 4093, 4096, 32003])
@pytest.mark.parametrize("entries", [1, 2, 3, 4])
def test_tables_on_any_boundary(vocab, entries):
    slots, rows = 3, 4
    g = torch.Generator().manual_seed(vocab)
    logits = torch.randn((rows, vocab), generator=g) * 4
    row_slot = torch.tensor([2, 0, 1, 2], dtype=torch.int32)
    tables = made(vocab, slots, vocab + entries, biases=min(9, vocab), grammar=True, known=0.4)
    device = LogitTables(**{name: moved(tensor, entries) for name, tensor in tables.items()})
    check(both_ways(logits, row_slot, device), logits, row_slot, tables, 2 + min(9, vocab))


def test_all_slots_but_the_first():
    """``counts[1:]`` of an odd vocabulary starts on no 16-byte boundary."""
    vocab = 32003
    tables = made(vocab, 4, 1, known=0.4)
    device = {name: tensor.to(DEVICE) for name, tensor in tables.items()}
    g = torch.Generator().manual_seed(2)
    logits, row_slot = torch.randn((3, vocab), generator=g), torch.tensor([2, 0, 1], dtype=torch.int32)
    view = LogitTables(**{name: tensor[1:] for name, tensor in device.items()})
    assert view.counts.data_ptr() % 16
    check(both_ways(logits, row_slot, view), logits, row_slot, {name: tensor[1:] for name, tensor in tables.items()}, 0)


@pytest.mark.parametrize("vocab", [1, 3, 5, 30, 33, 1000, 1021, 4093, 4097])
def test_bits_behind_the_vocabulary_say_nothing(vocab):
    """The last word of ``seen`` and ``allowed`` has bits for tokens that do not exist, set or not."""
    slots, rows = 3, 4
    g = torch.Generator().manual_seed(vocab)
    logits = torch.randn((rows, vocab), generator=g) * 4
    row_slot = torch.tensor([2, 0, 1, 2], dtype=torch.int32)      # the last slot's words end where the table ends
    tables = made(vocab, slots, vocab, grammar=True, known=0.6)
    filled = {name: tensor.to(DEVICE) for name, tensor in tables.items()}
    want = both_ways(logits, row_slot, LogitTables(**filled))
    if vocab % 32:
        behind = -1 << (vocab % 32)
        filled["seen"][:, -1] |= behind
        filled["allowed"][:, -1] ^= behind
    got = both_ways(logits, row_slot, LogitTables(**filled))
    assert torch.equal(got, want)
    check(got, logits, row_slot, tables, 0)
