"""``linear_adapters`` over many rows, where the adapters extend the shared product and the sums u = scale x A^T enter the tensor
cores in bfloat16 parts: float32 results keep the bits of u, and an infinite entry of B gives what the formula gives."""

from __future__ import annotations

import pytest
import torch

from mini_llm_runtime_b200 import ops
from test_adapters_gpu import check, made, run, some_ids

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


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,N,rank", [(4, 1152, 16), (40, 1152, 16), (200, 1152, 8), (300, 1152, 72), (1500, 1152, 16), (700, 9728, 72)])
def test_an_infinite_entry_of_b(rows, N, rank, out_dtype):
    """u B with one infinite entry in a column of B: infinite, with the sign of their product, at any number of rows; NaN where u is
    zero; every other column as the formula has it."""
    K = 128
    case = made(rows, K, N, rank, 3, torch.bfloat16, rows + rank)
    case["x"][1] = 0.0                                    # u = 0
    case["x"][2] = 0.0
    case["x"][2, 5], case["down"][:, :, 5], case["scales"][:] = 1.0, 0.5, 0.75       # u = 0.375: no bits behind the first part
    ids = some_ids(rows, 3, "one", 1)
    adapter = 2
    clean = run(case, ids, out_dtype)
    check(clean, case, ids, out_dtype)
    columns, ranks = [3, 200, N - 1], [0, rank - 1, rank // 2]
    kept = case["up"].clone()
    for column, r, sign in zip(columns, ranks, (1.0, -1.0, 1.0)):
        case["up"][adapter, column, r] = sign * float("inf")
    got = run(case, ids, out_dtype)
    u = (case["scales"][adapter].double() * case["x"].double() @ case["down"][adapter].double().T)
    for column, r, sign in zip(columns, ranks, (1.0, -1.0, 1.0)):
        want = u[:, r].sign() * sign * float("inf")       # NaN for u = 0
        # a sum of 128 products that is this close to zero could have either sign in 32 bits (none or one in a few thousand)
        near = (u[:, r].abs() <= 2.0 ** -17 * (case["x"].double().abs() @ case["down"][adapter, r].double().abs())) & (u[:, r] != 0)
        same = (got[:, column].double() == want) | (got[:, column].isnan() & want.isnan()) | near
        assert bool(same.all()), (column, torch.nonzero(~same).flatten().tolist()[:5])
    others = torch.ones(N, dtype=torch.bool, device=DEVICE)
    others[columns] = False
    assert torch.equal(got[:, others], clean[:, others])
    case["up"] = kept
    assert torch.equal(run(case, ids, out_dtype), clean)
