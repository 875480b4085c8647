"""A cache in 8 bits where calls follow one another, sizes are small and scales far apart: the edges of ``quantized_attention``."""

from __future__ import annotations

import copy

import numpy as np
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


@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(12, 3, 96, torch.float32), (20, 2, 64, torch.float32), (6, 2, 80, torch.bfloat16),
                                                      (14, 2, 64, torch.bfloat16), (8, 2, 128, torch.bfloat16), (20, 1, 64, torch.bfloat16)])
def test_a_value_without_number_counts_however_small_its_weight(heads, kv_heads, dim, dtype):
    """A seen key whose score lies so far below the others' that its weight is zero, its value's scale NaN: decoded tokens and a prompt's rows."""
    step = Step([1, 6, 1], [300, 90, 40], heads, kv_heads, dim, 16, 1, dtype, 70)
    step.q.abs_().clamp_(min=0.5)
    for i, at in ((0, 150), (1, 20)):
        page, offset = step.place(i, at + 1)
        page, offset = int(page[at]), int(offset[at])
        step.pool.key[page, :, offset] = -127
        step.pool.key_scales[page, :, offset] = 100.0
        step.pool.value_scales[page, :, offset] = float("nan")
    # With a number there, the weight is none: the rows are those of any other number.  In 32 bits to the last bit; the tensor cores' weights
    # carry the values' scales, of a prompt their largest power of two among 64 keys, which this one's scale is one of: weights in float16
    # are off by 2^-11 of their contributions, sum p |v| <= 2.1 here (scales up to 2.1 / 127), and, relative to a largest of at least one, by 2^-25
    # times a value of at most 254 steps of a scale of at most one, for each of n keys; each of the two results by half a step beside that.
    values, held = [], step.pool.value_scales.clone()
    for number in (0.0, 1.0):
        step.pool.value_scales.copy_(torch.where(held.isnan(), number, held))
        values.append(step.run())
    assert bool(torch.isfinite(values[0]).all())
    if dtype == torch.float32 or dim not in (64, 128):
        assert torch.equal(*values)
    else:
        zero, one = values[0].double(), values[1].double()
        allowed = torch.finfo(dtype).eps * torch.maximum(zero.abs(), one.abs()) + 2 * (2.0 ** -11 * 2.1 + 301 * 2.0 ** -25 * 254)
        assert bool(((zero - one).abs() <= allowed).all())
    step.pool.value_scales.copy_(held)
    got = step.run()
    assert bool(torch.isnan(got[:7]).all()) and torch.equal(got[7:], values[0][7:])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_places_that_no_key_is_seen_at_give_nothing(dtype):
    """Beside them in a tile: keys before the window and behind the row, their scales not finite."""
    step = Step([1, 1], [300, 70], 12, 3, 96, 16, 1, dtype, 71)
    want = step.run(window=50)
    for i, seen in ((0, range(251, 301)), (1, range(21, 71))):
        page, offset = step.place(i, int(step.first[i]) // 16 * 16 + 16)
        for at in set(range(len(page))) - set(seen):
            step.pool.value_scales[page[at], :, offset[at]] = float("inf" if at % 2 else "nan")
    assert torch.equal(step.run(window=50), want)


def rows_before(step, i, rows):
    """The step's request i as if it had only its first ``rows`` rows, and where these lie in the step."""
    short = copy.copy(step)
    at = int(step.start[i])
    short.lengths, short.first, short.slots, short.start = (np.asarray([rows], dtype=np.int32), step.first[i:i + 1], step.slots[i:i + 1],
                                                            np.zeros(1, dtype=np.int32))
    short.q = step.q[at:at + rows]
    return short, slice(at, at + rows)


@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(14, 2, 64, torch.bfloat16), (8, 2, 128, torch.bfloat16), (12, 3, 96, torch.float32)])
@pytest.mark.parametrize("which", ["keys", "values", "both"])
@pytest.mark.parametrize("power", [5, 7, 30, 60])
def test_scales_of_later_keys_do_not_reach_the_rows_before_them(heads, kv_heads, dim, dtype, which, power):
    """Rows of a prompt whose later keys' scales are larger by far, in the same 64 keys and behind: held to the errors of what they see."""
    step = Step([100, 1, 40], [70, 33, 0], heads, kv_heads, dim, 16, 1, dtype, 80)
    for i, cut in ((0, 95), (2, 21)):      # positions from which on
        page, offset = step.place(i, int(step.first[i] + step.lengths[i]))
        for name, scales in (("keys", step.pool.key_scales), ("values", step.pool.value_scales)):
            if which in (name, "both"):
                scales[page[cut:], :, offset[cut:]] *= 2.0 ** power
    got = step.run()
    for i, cut in ((0, 95), (2, 21)):
        short, rows = rows_before(step, i, cut - int(step.first[i]))
        short.check(got[rows])
    short, rows = rows_before(step, 1, 1)
    short.check(got[rows])


@pytest.mark.parametrize("heads,kv_heads,dim", [(14, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("key,value,query", [(1e-20, 1.0, 1e-30), (1.0, 1e-25, 1.0), (1e-25, 1e-25, 1.0), (1e6, 1e-6, 1e-6), (1e-12, 1e20, 1e12)])
def test_scales_and_queries_far_from_one(heads, kv_heads, dim, key, value, query):
    step = Step([1, 90, 1, 3], [100, 30, 3, 500], heads, kv_heads, dim, 16, 4, torch.bfloat16, 81)
    step.pool.key_scales.mul_(key)
    step.pool.value_scales.mul_(value)
    step.q.mul_(query)
    step.check(step.run())


@pytest.mark.parametrize("heads,kv_heads,dim", [(14, 2, 64), (8, 2, 128)])
def test_scales_of_one_request_further_apart_than_float16_is_wide(heads, kv_heads, dim):
    """Every key with a power of two of its own between 2^-30 and 1, a tenth of the blocks zeros: each key by itself, over several tiles, windows too."""
    step = Step([1, 150, 1, 64], [300, 100, 7, 1000], heads, kv_heads, dim, 16, 1, torch.bfloat16, 82)
    g = torch.Generator(device=DEVICE).manual_seed(83)
    for scales, codes in ((step.pool.value_scales, step.pool.value), (step.pool.key_scales, step.pool.key)):
        scales *= 2.0 ** torch.randint(-30, 1, scales.shape, generator=g, device=DEVICE).float()
        empty = torch.rand(scales.shape, generator=g, device=DEVICE) < 0.1
        scales[empty] = 0.0
        codes.view(*scales.shape, -1, dim)[empty] = 0
    step.check(step.run())
    step.check(step.run(window=40), window=40)
