"""``linear_adapters`` over many rows, where the adapters extend the shared product and the sums u = scale x A^T enter the tensor
cores in bfloat16 parts: float32 results keep the bits of u."""

from __future__ import annotations

import pytest
import torch

from mini_llm_runtime_b200 import ops
from mini_llm_runtime_b200.ops import AdapterStack
from test_adapters_gpu import made, run, some_ids

pytestmark = pytest.mark.gpu

DEVICE = "cuda:0"


# the third and fifth: tiles of 128 x 256 with rings of two stages, which hold two parts of u at a time; the last: 256 x 256
@pytest.mark.parametrize("rows,K,N,rank", [(200, 64, 520, 8), (300, 256, 264, 24), (1000, 128, 8000, 72), (150, 64, 1000, 128), (1500, 64, 9728, 16),
                                           (1500, 2048, 4608, 72)])
def test_a_float32_result_has_all_of_u(rows, K, N, rank):
    """One product per result: W is zero, a row of x has one entry and B one rank for each column, so y = scale x A B.  u is rounded
    once (2^-24); each of its parts meets B in an exact product, and a sum of a part with what stands in the accumulator is off by
    at most 2^-22 of it (cut off behind 23 bits, of two terms): 2^-24 + 3 * 2^-22 < 2^-20 of y."""
    g = torch.Generator(device=DEVICE).manual_seed(rows)
    case = made(rows, K, N, rank, 3, torch.bfloat16, rows, bias=False)
    case["weight"].zero_()
    place = torch.randint(0, K, (rows,), generator=g, device=DEVICE)
    case["x"] *= torch.nn.functional.one_hot(place, K)
    column = torch.randint(0, rank, (N,), generator=g, device=DEVICE)
    case["up"] *= torch.nn.functional.one_hot(column, rank)
    ids = some_ids(rows, 3, "runs", 1)
    kernels = ops.current()
    assert kernels._adapters_extend(rows, N, K, rank)
    got = run(case, ids, torch.float32)
    for adapter in range(3):
        mine = torch.nonzero(ids == adapter).flatten()
        u = float(case["scales"][adapter]) * case["x"][mine].double() @ case["down"][adapter].double().T
        want = u @ case["up"][adapter].double().T
        assert bool(((got[mine].double() - want).abs() <= 2.0 ** -20 * want.abs()).all())
    assert not bool(got[ids < 0].any())
