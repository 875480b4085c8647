"""Attention over keys and values in 8 bits (``quantized_attention``) against softmax attention in 64 bits over what the codes stand for."""

from __future__ import annotations

import pytest
import torch

from mini_llm_runtime_b200 import ops
from quantized_support import Step

pytestmark = pytest.mark.gpu

DEVICE = "cuda:0"

SHAPES = [
    # heads, kv_heads, dim, page, block, dtype
    (14, 2, 64, 16, 16, torch.bfloat16), (28, 4, 128, 16, 16, torch.bfloat16), (40, 8, 128, 16, 1, torch.bfloat16),
    (16, 1, 128, 32, 4, torch.bfloat16), (4, 4, 64, 8, 8, torch.bfloat16), (16, 16, 64, 64, 64, torch.bfloat16), (12, 3, 96, 16, 4, torch.float32),
    (6, 2, 80, 16, 16, torch.bfloat16), (14, 2, 64, 5, 5, torch.bfloat16), (2, 1, 256, 16, 2, torch.float32), (3, 1, 17, 6, 3, torch.float32),
    (20, 1, 64, 16, 16, torch.bfloat16), (14, 2, 64, 128, 32, torch.float32), (8, 2, 128, 256, 256, torch.bfloat16)]


@pytest.mark.parametrize("heads,kv_heads,dim,page,block,dtype", SHAPES)
def test_decoded_tokens(heads, kv_heads, dim, page, block, dtype):
    first = [0, 1, page - 1, page, 31, 32, 33, 63, 64, 127, 200, 777]
    step = Step([1] * len(first), first, heads, kv_heads, dim, page, block, dtype, 1)
    step.check(step.run())


@pytest.mark.parametrize("heads,kv_heads,dim,page,block,dtype", SHAPES)
def test_prompt_portions_beside_decoded_tokens(heads, kv_heads, dim, page, block, dtype):
    step = Step([5, 1, 130, 1, 2, 17, 1], [0, 70, 40, 0, 300, 16, 129], heads, kv_heads, dim, page, block, dtype, 2)
    step.check(step.run())


@pytest.mark.parametrize("heads,kv_heads,dim,page,block,dtype", SHAPES[:9])
@pytest.mark.parametrize("window", [1, 40, 64])
def test_windows(heads, kv_heads, dim, page, block, dtype, window):
    step = Step([1, 1, 1, 90, 3, 1], [0, 39, 500, 100, 64, 63], heads, kv_heads, dim, page, block, dtype, 3)
    step.check(step.run(window=window), window=window)


@pytest.mark.parametrize("heads,kv_heads,dim,page,block,dtype", SHAPES[:4])
def test_long_contexts(heads, kv_heads, dim, page, block, dtype):
    step = Step([1, 1, 1], [9000, 4095, 12345], heads, kv_heads, dim, page, block, dtype, 4)
    step.check(step.run())


@pytest.mark.parametrize("heads,kv_heads,dim,page,block,dtype", SHAPES[:3])
def test_many_requests(heads, kv_heads, dim, page, block, dtype):
    step = Step([1] * 200, [(i * 37) % 400 for i in range(200)], heads, kv_heads, dim, page, block, dtype, 5)
    step.check(step.run())


@pytest.mark.parametrize("heads,kv_heads,dim,page,block,dtype", SHAPES[:2])
def test_long_prompts(heads, kv_heads, dim, page, block, dtype):
    step = Step([700, 1, 129], [1000, 50, 0], heads, kv_heads, dim, page, block, dtype, 6)
    step.check(step.run())


@pytest.mark.parametrize("heads,kv_heads,dim,page,block,dtype", [SHAPES[0], SHAPES[1], SHAPES[2], SHAPES[6]])
def test_scales_of_many_sizes(heads, kv_heads, dim, page, block, dtype):
    """Values whose scales differ by powers of two, keys likewise; blocks of zeros, their scale zero."""
    step = Step([1, 1, 60, 1], [100, 900, 40, 3], heads, kv_heads, dim, page, block, dtype, 7)
    g = torch.Generator(device=DEVICE).manual_seed(8)
    for scales, codes in ((step.pool.value_scales, step.pool.value), (step.pool.key_scales, step.pool.key)):
        scales *= 2.0 ** torch.randint(-6, 2, scales.shape, generator=g, device=DEVICE).float()
        empty = torch.rand(scales.shape, generator=g, device=DEVICE) < 0.1
        scales[empty] = 0.0
        codes.view(*scales.shape, -1, dim)[empty] = 0
    step.check(step.run())


@pytest.mark.parametrize("heads,kv_heads,dim,page,block,dtype", [SHAPES[0], SHAPES[1], SHAPES[2], SHAPES[6], SHAPES[7]])
def test_what_lies_in_places_that_a_row_does_not_see(heads, kv_heads, dim, page, block, dtype):
    """NaN and infinite scales behind the last key, on pages of nobody, and (a block of one token) at later positions of a prompt."""
    step = Step([1, 40, 1], [20, 33, 130], heads, kv_heads, dim, page, block, dtype, 9)
    want = step.run()
    used = torch.zeros(step.pool.pages, page // block, dtype=torch.bool, device=DEVICE)
    for i in range(3):
        pages, offsets = step.place(i, int(step.first[i] + step.lengths[i]))
        used[pages, offsets // block] = True
    for scales, bad in ((step.pool.key_scales, float("nan")), (step.pool.value_scales, float("inf"))):
        scales[~used[:, None].expand_as(scales)] = bad
    assert torch.equal(step.run(), want)
    if block == 1:
        page_of, offset = step.place(1, 73)
        for scales, bad in ((step.pool.key_scales, float("nan")), (step.pool.value_scales, float("nan"))):
            scales[page_of[60], :, offset[60]] = bad
        got = step.run()
        assert torch.equal(got[:28], want[:28]) and torch.equal(got[41:], want[41:])       # rows of positions 33 .. 59, the other requests
        assert bool(torch.isnan(got[28:41]).all())


def test_no_row_and_what_is_refused():
    step = Step([1, 3], [20, 33], 14, 2, 64, 16, 16, torch.bfloat16, 10)
    batch, k = step.batch(), ops.current()
    assert k.quantized_attention(step.q[:0], step.pool, batch, 14, 2, 64, 0.125).shape == (0, 14 * 64)
    for call in (lambda: k.quantized_attention(step.q, step.pool, batch, 14, 4, 64, 0.125),
                 lambda: k.quantized_attention(step.q, step.pool, batch, 7, 2, 128, 0.125),
                 lambda: k.quantized_attention(step.q, step.pool, batch, 15, 2, 64, 0.125),
                 lambda: k.quantized_attention(step.q.half(), step.pool, batch, 14, 2, 64, 0.125),
                 lambda: k.quantized_attention(step.q.cpu(), step.pool, batch, 14, 2, 64, 0.125),
                 lambda: k.quantized_attention(step.q.t().contiguous().t(), step.pool, batch, 14, 2, 64, 0.125)):
        with pytest.raises(ops.KernelError):
            call()


@pytest.mark.parametrize("heads,kv_heads,dim,page,block,dtype", [SHAPES[0], SHAPES[1], SHAPES[6]])
def test_calls_side_by_side_and_two_graphs(heads, kv_heads, dim, page, block, dtype):
    """Steps on two streams at once, eager and captured, share no memory of theirs: prompts whose keys are cut into parts beside decoded tokens."""
    steps = [Step([300, 1, 40, 1], [900 + 500 * i, 700, 100, 1300], heads, kv_heads, dim, page, block, dtype, 20 + i) for i in range(2)]
    batches = [step.batch() for step in steps]
    want = [step.run() for step in steps]
    for step, alone in zip(steps, want):
        step.check(alone)
    call = lambda i: ops.current().quantized_attention(steps[i].q, steps[i].pool, batches[i], heads, kv_heads, dim, steps[i].scale)
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    got, graphs, captured = [[], []], [], []
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(call(i))
    torch.cuda.synchronize()
    for i, stream in enumerate(streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            captured.append(call(i))
        graphs.append(graph)
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    ops.current().raise_if_device_error()
    for i in range(2):
        for one in (*got[i], captured[i]):
            assert torch.equal(one, want[i])
