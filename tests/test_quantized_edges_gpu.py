"""A cache in 8 bits where calls follow one another, sizes are small and scales far apart: the edges of ``quantized_attention``."""

from __future__ import annotations

import pytest
import torch

from mini_llm_runtime_b200 import ops
from quantized_support import Step

pytestmark = pytest.mark.gpu

DEVICE = "cuda:0"


@pytest.mark.parametrize("heads,kv_heads,dim", [(14, 2, 64), (8, 2, 128)])
def test_prompts_of_other_sizes_one_behind_the_other_on_one_stream(heads, kv_heads, dim, monkeypatch):
    """A call's memory is the last one's while that still runs: few rows behind many keys, then several short prompts, then decoded tokens between
    two portions, whose tiles begin at other places of the same block."""
    shapes = [([9], [6000]), ([40, 3, 17, 130], [1500, 2700, 0, 900]), ([5, 1, 1, 33], [900, 50, 70, 4300]), ([2, 2], [0, 3000])]
    steps = [Step(lengths, first, heads, kv_heads, dim, 16, 16, torch.bfloat16, 40 + i) for i, (lengths, first) in enumerate(shapes)]
    batches = [step.batch() for step in steps]
    call = lambda i: ops.current().quantized_attention(steps[i].q, steps[i].pool, batches[i], heads, kv_heads, dim, steps[i].scale)
    want = []
    for i, step in enumerate(steps):
        want.append(call(i))
        torch.cuda.synchronize()
        step.check(want[i])
    # what torch's allocator may do with memory that a call has given back: every call's begins at one place
    arena, taken, empty = torch.empty(64 << 20, dtype=torch.uint8, device=DEVICE), [0], torch.empty

    def within(*args, **kwargs):
        if kwargs.get("dtype") != torch.uint8:
            return empty(*args, **kwargs)
        begin = taken[0]
        taken[0] = (begin + int(args[0]) + 511) // 512 * 512
        return arena[begin:begin + int(args[0])]

    monkeypatch.setattr(torch, "empty", within)
    got = []
    for turn in range(40):
        for i in range(len(steps)):
            taken[0] = 0
            got.append((i, call(i)))
    monkeypatch.undo()
    torch.cuda.synchronize()
    ops.current().raise_if_device_error()
    assert 0 < taken[0] <= arena.numel()
    for i, one in got:
        assert torch.equal(one, want[i])


@pytest.mark.parametrize("dim", [1, 2, 3, 4, 5, 8, 12])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (4, 1), (3, 1), (10, 2), (9, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decoded_tokens_of_small_heads(heads, kv_heads, dim, dtype):
    """Heads of so few dimensions that a thread block has more threads than a tile's keys times a row's pieces."""
    first = [0, 1, 15, 16, 63, 64, 65, 255, 256, 700]
    step = Step([1] * len(first), first, heads, kv_heads, dim, 16, 4, dtype, 50 + dim)
    step.check(step.run())
    step = Step([5, 1, 30, 1], [0, 70, 40, 600], heads, kv_heads, dim, 16, 16, dtype, 60 + dim)
    step.check(step.run())
