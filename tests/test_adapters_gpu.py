"""A projection with the low-rank adapters of many requests (``linear_adapters``) against its formula in 64 bits, row by row: ranks
and widths that no tile divides, one adapter for all rows, one for each, rows without one, ids outside the stack."""

from __future__ import annotations

import pytest
import torch

from mini_llm_runtime_b200 import ops
from mini_llm_runtime_b200.ops import AdapterStack

pytestmark = pytest.mark.gpu

DEVICE = "cuda:0"


def made(rows, K, N, rank, count, dtype, seed, bias=True):
    g = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device=DEVICE) * scale).to(dtype)

    return dict(x=normal(rows, K), weight=normal(N, K, scale=K ** -0.5), bias=normal(N) if bias else None,
                down=normal(count, rank, K, scale=K ** -0.5), up=normal(count, N, rank, scale=rank ** -0.5),
                scales=torch.rand(count, generator=g, device=DEVICE) * 2 - 0.5)


def check(got, case, ids, out_dtype):
    """|error| <= half a step of the result's type, plus the sums' roundings in 32 bits: of n products of total magnitude S
    rounded n times to 24 bits at most 4 sqrt(n) 2^-24 S for roundings that are not all of one sign, or, cut off instead of
    rounded every 16 products, n / 16 times 2^-23 of a running sum of about S / sqrt(n); and u in two bfloat16 parts, 2^-16."""
    x, weight = case["x"].double(), case["weight"].double()
    want = x @ weight.T
    size = x.abs() @ weight.abs().T
    low_size = torch.zeros_like(size)
    if case["bias"] is not None:
        want += case["bias"].double()
        size += case["bias"].double().abs()
    count, rank = case["down"].shape[:2]
    for adapter in range(count):
        rows = torch.nonzero(ids == adapter).flatten()
        if len(rows):
            down, up, scale = case["down"][adapter].double(), case["up"][adapter].double(), float(case["scales"][adapter])
            want[rows] += scale * (x[rows] @ down.T) @ up.T
            low_size[rows] += abs(scale) * (x[rows].abs() @ down.abs().T) @ up.abs().T
    K = x.shape[1]
    bound = torch.finfo(out_dtype).eps / 2 * want.abs() + 4 * K ** 0.5 * 2.0 ** -24 * (size + low_size) * 1.01 + 2.0 ** -16 * low_size
    worst = ((got.double() - want).abs() - bound).max()
    assert torch.isfinite(got).all()
    assert float(worst) <= 0, float(worst)


def run(case, ids, out_dtype=None):
    stack = AdapterStack(case["down"], case["up"], case["scales"])
    return ops.current().linear_adapters(case["x"], case["weight"], stack, ids, bias=case["bias"], out_dtype=out_dtype)


def some_ids(rows, count, pattern, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    if pattern == "one":
        ids = torch.full((rows,), count - 1, device=DEVICE)
    elif pattern == "none":
        ids = torch.full((rows,), -1, device=DEVICE)
    elif pattern == "runs":
        ids = torch.arange(rows, device=DEVICE) * 5 // max(1, rows) % (count + 1) - 1
    else:      # mixed: every adapter, none, and ids outside the stack
        ids = torch.randint(-2, count + 2, (rows,), generator=g, device=DEVICE)
    return ids.to(torch.int32)


@pytest.mark.parametrize("pattern", ["one", "none", "runs", "mixed"])
@pytest.mark.parametrize("rows,K,N,rank,count", [
    (1, 8, 8, 1, 1), (1, 896, 1152, 8, 4), (3, 100, 37, 5, 3), (7, 256, 136, 16, 4), (16, 520, 264, 24, 9), (33, 1000, 200, 64, 3),
    (1, 16, 5, 128, 2), (2, 128, 72, 16, 4), (3, 64, 41, 7, 5), (4, 40, 100, 33, 6), (2, 896, 1152, 8, 3), (64, 896, 520, 12, 40), (130, 640, 392, 32, 6), (257, 384, 1000, 128, 7), (300, 72, 264, 40, 5),
])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_adapters_against_their_formula(dtype, rows, K, N, rank, count, pattern):
    case = made(rows, K, N, rank, count, dtype, rows + K)
    ids = some_ids(rows, count, pattern, rows)
    check(run(case, ids), case, ids, dtype)
    if dtype == torch.bfloat16:
        check(run(case, ids, torch.float32), case, ids, torch.float32)


@pytest.mark.parametrize("rows,K,N,rank,count,pattern", [
    (600, 896, 2048, 16, 5, "runs"), (1025, 512, 1160, 64, 3, "mixed"), (513, 2048, 4608, 48, 20, "runs"),
    (2048, 1024, 3584, 8, 2, "runs"), (700, 640, 776, 128, 600, "mixed"),
    (17, 640, 15880, 128, 3, "runs"), (40, 896, 9728, 128, 50, "mixed"), (128, 200, 4608, 64, 2, "one"),
])
def test_prompt_steps(rows, K, N, rank, count, pattern):
    case = made(rows, K, N, rank, count, torch.bfloat16, rows, bias=rows % 2 == 1)
    ids = some_ids(rows, count, pattern, 3)
    check(run(case, ids), case, ids, torch.bfloat16)


def test_rows_without_an_adapter_are_the_shared_product():
    case = made(40, 256, 128, 8, 2, torch.float32, 5)
    ids = some_ids(40, 2, "none", 1)
    assert torch.equal(run(case, ids), ops.current().linear(case["x"], case["weight"], case["bias"]))


def test_no_rows():
    case = made(0, 64, 32, 8, 2, torch.bfloat16, 5)
    assert run(case, torch.empty(0, dtype=torch.int32, device=DEVICE)).shape == (0, 32)


@pytest.mark.parametrize("rows", [2, 20, 300])
def test_an_infinite_sum_stays_infinite(rows):
    """x A^T infinite and B positive: infinity, not the NaN of an infinity taken from itself; the other rows are what they were."""
    case = made(rows, 128, 1152, 16, 2, torch.bfloat16, 8)
    ids = some_ids(rows, 2, "one", 1)
    want = run(case, ids)
    case["x"][1, 0] = float("inf")
    case["weight"][:, 0], case["down"][:, :, 0], case["up"][:], case["scales"][:] = 0.5, 0.25, 0.125, 1.0
    got = run(case, ids)
    assert (got[1] == float("inf")).all()
    case["x"][1, 0] = 0.0
    again = run(case, ids)
    others = torch.arange(rows, device=DEVICE) != 1
    assert torch.equal(got[others], again[others]) and torch.isfinite(want).all()


def test_what_other_adapters_hold_does_not_matter():
    """Infinities and NaN in adapters that no row of the batch uses, and in the rows of x that use none."""
    case = made(20, 128, 264, 16, 4, torch.bfloat16, 6)
    ids = some_ids(20, 2, "runs", 1)
    want = run(case, ids)
    case["down"][2:], case["up"][2:], case["scales"][2:] = float("nan"), float("inf"), float("nan")
    assert torch.equal(run(case, ids), want)
    many = made(300, 128, 264, 16, 4, torch.bfloat16, 7)
    ids = some_ids(300, 2, "runs", 1)
    want = run(many, ids)
    many["down"][2:], many["up"][2:], many["scales"][2:] = float("nan"), float("inf"), float("nan")
    assert torch.equal(run(many, ids), want)


@pytest.mark.parametrize("rows", [6, 300])
def test_a_row_not_finite_stays_alone(rows):
    case = made(rows, 128, 264, 16, 4, torch.bfloat16, 8)
    ids = some_ids(rows, 4, "runs", 1)
    want = run(case, ids)
    case["x"][rows // 2, 3] = float("inf")
    got = run(case, ids)
    others = torch.arange(rows, device=DEVICE) != rows // 2
    assert torch.equal(got[others], want[others])
    assert not bool(torch.isfinite(got[rows // 2]).all())


@pytest.mark.parametrize("rows,rank", [(6, 16), (60, 8), (300, 16), (300, 128), (300, 12)])
def test_an_adapter_not_finite_stays_with_its_rows(rows, rank):
    case = made(rows, 128, 264, rank, 4, torch.bfloat16, 8)
    ids = some_ids(rows, 4, "mixed", 1)
    want = run(case, ids)
    case["down"][1], case["up"][2] = float("inf"), float("nan")
    got = run(case, ids)
    others = (ids != 1) & (ids != 2)
    assert torch.equal(got[others], want[others])
    assert not bool(torch.isfinite(got[~others]).any())


@pytest.mark.parametrize("rows", [5, 280])
def test_a_captured_projection_follows_its_adapters(rows):
    case = made(rows, 256, 512, 16, 6, torch.bfloat16, 9)
    ids = some_ids(rows, 6, "mixed", 1)
    run(case, ids)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(case, ids)
    for turn in range(3):
        ids.copy_(some_ids(rows, 6, "mixed" if turn else "one", turn + 7))
        case["x"].copy_(torch.randn_like(case["x"]))
        graph.replay()
        torch.cuda.synchronize()
        check(out, case, ids, torch.bfloat16)


def test_repeated_calls_give_the_same_bits():
    for rows in (9, 290):
        case = made(rows, 1000, 520, 24, 6, torch.bfloat16, 10)
        ids = some_ids(rows, 6, "mixed", 2)
        first = run(case, ids)
        for _ in range(5):
            assert torch.equal(run(case, ids), first)


def test_on_another_stream():
    case = made(12, 256, 512, 16, 6, torch.bfloat16, 11)
    ids = some_ids(12, 6, "mixed", 2)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = run(case, ids)
    stream.synchronize()
    check(got, case, ids, torch.bfloat16)


def test_a_stack_of_more_than_32_bit_offsets():
    count, rank, K, N = 130, 128, 131072, 8         # 2.2e9 entries in down
    g = torch.Generator(device=DEVICE).manual_seed(1)
    down = torch.zeros((count, rank, K), dtype=torch.bfloat16, device=DEVICE)
    down[count - 1] = torch.randn((rank, K), generator=g, device=DEVICE).to(torch.bfloat16) * K ** -0.5
    case = made(2, K, N, rank, 1, torch.bfloat16, 12)
    case["down"], case["up"] = down, torch.randn((count, N, rank), generator=g, device=DEVICE).to(torch.bfloat16)
    case["scales"] = torch.ones(count, device=DEVICE)
    ids = torch.tensor([count - 1, -1], dtype=torch.int32, device=DEVICE)
    got = run(case, ids)
    small = {**case, "down": down[count - 1:], "up": case["up"][count - 1:], "scales": case["scales"][count - 1:]}
    check(got, small, torch.tensor([0, -1], device=DEVICE), torch.bfloat16)


@pytest.mark.parametrize("rows", [1, 20, 200])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_weight_on_no_16_byte_boundary(dtype, rows):
    case = made(rows, 256, 264, 16, 4, dtype, 13)
    buffer = torch.empty(264 * 256 + 1, dtype=dtype, device=DEVICE)
    buffer[1:] = case["weight"].flatten()
    case["weight"] = buffer[1:].view(264, 256)
    ids = some_ids(rows, 4, "mixed", 2)
    check(run(case, ids), case, ids, dtype)


def test_x_on_no_16_byte_boundary_is_refused():
    case = made(3, 64, 40, 8, 2, torch.bfloat16, 14)
    case["x"] = torch.zeros(3 * 64 + 1, dtype=torch.bfloat16, device=DEVICE)[1:].view(3, 64)
    with pytest.raises(ops.KernelError, match="boundary"):
        run(case, some_ids(3, 2, "one", 1))


def test_without_the_tensor_cores(monkeypatch):
    """The switch that keeps products on the CUDA cores."""
    monkeypatch.setattr(ops.current(), "use_tensor_cores", False)
    for rows in (5, 40, 200):
        case = made(rows, 256, 264, 16, 4, torch.bfloat16, 15)
        ids = some_ids(rows, 4, "mixed", 2)
        check(run(case, ids), case, ids, torch.bfloat16)
